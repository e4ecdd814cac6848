"""The decoder's own prefill -- whole prompts packed, and one prompt in chunks over a paged cache -- and its dense layers over
a paged cache, run together as a server would: prefill, decode steps, captured graph."""
import pytest
import torch

from magicpig_amd import decode_harness as dh

SHAPE = dict(num_hidden_layers=3, num_attention_heads=4, num_key_value_heads=2, intermediate_size=768, vocab_size=1000)
# A layer rounds its activations to bf16 at most 14 times between its input and output (norms, projections, rotation, attention
# and its weights, gate, residual sums), each by 2^-8 of the value at most, and three layers and the head pass errors on with gains of
# about 1 (weights are drawn that way): logits of two runs that round at different places differ by less than
BOUND = (3 * 14 + 4) * 2.0 ** -8


def decoder(head_dim=128, **kw):
    shape = dh.LlamaShape(hidden_size=4 * head_dim, **SHAPE)
    # one bit a table: practically every offloaded token is sampled, the sparse layers attend to everything
    kw = {**dict(K=1, L=64, batch_size=2, max_length=1024, generation_buffer=16, dense_layers=(0,), seed=3), **kw}
    return dh.SyntheticLlamaDecoder(shape, **kw)


def prompts(*lens):
    g = torch.Generator().manual_seed(1)
    return [torch.randint(0, 1000, (n,), generator=g).cuda() for n in lens]


def close(a, b, bound=BOUND):
    a, b = a.double(), b.double()
    off = ((a - b).norm(dim=-1) / b.norm(dim=-1)).max().item()
    assert off < bound, f"logits differ by {off:.4f} of their norm, bound {bound:.4f}"


def reference_prefill(dec, ids):
    """The model in f32 on one prompt, attention written out."""
    H, Hkv, D = 4, 2, dec._head_dim
    n, eps = ids.numel(), dec.shape.rms_norm_eps
    x = dec.embed_tokens[ids].float()

    def norm(y, w):
        return y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps) * w.float()

    def rope(y):
        ang = torch.arange(n, device="cuda")[:, None, None] * dec.shape.rope_theta ** (-torch.arange(D // 2, device="cuda").float() * 2 / D)
        a, b = y[..., :D // 2], y[..., D // 2:]
        return torch.cat((a * ang.cos() - b * ang.sin(), b * ang.cos() + a * ang.sin()), -1)

    for W in dec.layers:
        y = norm(x, W["ln1"])
        q, k, v = (y @ W[m].float().t() for m in ("wq", "wk", "wv"))
        q, k, v = rope(q.view(n, H, D)), rope(k.view(n, Hkv, D)), v.view(n, Hkv, D)
        outs = []
        for h in range(H):
            s = q[:, h] @ k[:, h * Hkv // H].t() / D ** 0.5
            s = s.masked_fill(torch.ones(n, n, device="cuda", dtype=torch.bool).triu(1), float("-inf"))
            outs.append(s.softmax(-1) @ v[:, h * Hkv // H])
        x = x + torch.cat(outs, -1) @ W["wo"].float().t()
        y = norm(x, W["ln2"])
        x = x + (torch.nn.functional.silu(y @ W["gate"].float().t()) * (y @ W["up"].float().t())) @ W["down"].float().t()
    return norm(x[-1:], dec.norm_weight) @ dec.lm_head.float().t()


@pytest.mark.gpu
@pytest.mark.parametrize("head_dim", [64, 128])
def test_packed_prefill_is_the_model(head_dim):
    dec = decoder(head_dim)
    ps = prompts(300, 71)
    logits = dec.prefill(ps)
    for i, p in enumerate(ps):
        close(logits[i:i + 1], reference_prefill(dec, p))
    assert dec.dense_len.tolist() == [300, 71]


@pytest.mark.gpu
@pytest.mark.parametrize("chunk", [1000, 128, 97])
@pytest.mark.parametrize("dense_cache", ["store", "bf16"])
def test_chunked_prefill_and_decode_follow_the_packed_one(chunk, dense_cache):
    a, b = decoder(), decoder(dense_cache=dense_cache)
    ps = prompts(500, 333)
    la = a.prefill(ps)
    for r, p in enumerate(ps):
        close(b.prefill_chunked(r, p, chunk=chunk), la[r:r + 1])
    ids = la.argmax(-1, keepdim=True)
    for step in range(3):
        pos = torch.tensor([[500 + step], [333 + step]], device="cuda")
        la, lb = a.inference(ids, pos), b.inference(ids, pos)
        close(lb, la)
        ids = la[:, -1].argmax(-1, keepdim=True)
    b.attention_server.window_server.check()
    b.dense_server.check()


@pytest.mark.gpu
def test_quantised_caches_stay_near():
    """e4m3 rounds keys and values by 2^-4 at most, 2^-5 on average of the worst place in a step: with weights that sum to 1 the
    attention output and the logits of keys move by no more than a few times that."""
    a, b = decoder(dense_layers=(0, 1, 2)), decoder(dense_layers=(0, 1, 2), dense_cache="e4m3")
    ps = prompts(400, 130)
    la = a.prefill(ps)
    for r, p in enumerate(ps):
        close(b.prefill_chunked(r, p, chunk=150, kv_format="e4m3"), la[r:r + 1], bound=BOUND + 3 * 2.0 ** -4)
    ids, pos = la.argmax(-1, keepdim=True), torch.tensor([[400], [130]], device="cuda")
    close(b.inference(ids, pos), a.inference(ids, pos), bound=BOUND + 4 * 2.0 ** -4)


@pytest.mark.gpu
def test_prefill_leaves_the_state_of_a_prompt_whose_cache_is_given():
    """The stores, tables and windows after prefill are those of prefill_synthetic given the same keys and values: decode
    steps agree bit for bit."""
    a, b = decoder(), decoder(dense_cache="bf16")
    kept = {}
    store = a._store_prompt
    a._store_prompt = lambda layer, r, k, v: (kept.__setitem__((layer, r), (k.clone(), v.clone())), store(layer, r, k, v))[1]
    ps = prompts(256, 700)
    la = a.prefill(ps, request_ids=[1, 0])
    c = decoder()
    for r, n in ((1, 256), (0, 700)):
        c.prefill_synthetic(r, n, kv=lambda layer, r=r: kept[(layer, r)])
        b.prefill_synthetic(r, n, kv=lambda layer, r=r: kept[(layer, r)])
    ids = la.argmax(-1, keepdim=True).flip(0)
    pos = torch.tensor([[700], [256]], device="cuda")
    x, y, z = (d.inference(ids, pos) for d in (a, c, b))
    assert torch.equal(x, y)
    close(z, x)


@pytest.mark.gpu
@pytest.mark.parametrize("dense_cache", ["bf16", "e4m3"])
def test_decode_loop_in_a_graph_over_pages(dense_cache):
    dec = decoder(dense_cache=dense_cache)
    ms, tps = dh.run_decode_benchmark(dec, 300, warmup=2, steps=4)
    assert ms > 0 and tps > 0 and dec.dense_len.tolist() == [300 + 2 + 2 + 4] * 2
    assert set(dh.split_decode_step(dec, reps=2)) == {"sparse_attention", "dense_attention", "projections_mlp", "norms_rope_residual", "embed_lm_head"}


@pytest.mark.gpu
def test_refusals():
    dec = decoder()
    ok = prompts(200)[0]
    for call in (lambda: dec.prefill([]), lambda: dec.prefill([ok, ok], request_ids=[0, 0]), lambda: dec.prefill([ok], request_ids=[2]),
                 lambda: dec.prefill([ok[:68]]), lambda: dec.prefill([prompts(1025)[0]]), lambda: dec.prefill_chunked(0, ok, chunk=0),
                 lambda: dec.prefill_chunked(-1, ok), lambda: dec.prefill_chunked(0, ok, kv_format="fp4")):
        with pytest.raises(ValueError):
            call()


def test_unknown_dense_cache_is_refused():
    with pytest.raises(ValueError, match="dense_cache"):
        dh.SyntheticLlamaDecoder(dense_cache="int4")
