"""The decoder's own prefill -- whole prompts packed, and one prompt in chunks over a paged cache -- and its dense layers over
a paged cache, run together as a server would: prefill, decode steps, captured graph."""
import pytest
import torch

import attention64
from magicpig_amd import decode_harness as dh
from magicpig_amd import MagicPigError
from test_gpu_paged_cache import stored

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


# ---------------------------------------------------------------- layer by layer: attention to its own roundings
def record(dec):
    """Everything that passes through the decoder's attention: prompt layers (layer, hidden, q, k, v, out, hidden out), rows that
    enter the state (layer, request): (k, v), dense decode layers (layer, q, k, v, out)."""
    log, rows, steps = [], {}, []
    layer_of, store, dense = dec._prompt_layer, dec._store_prompt, dec._dense_attention

    def prompt_layer(layer, hidden, pos, attend):
        kept = []

        def watched(q, k, v):
            out = attend(q, k, v)
            kept.extend(x.clone() for x in (q, k, v, out))
            return out
        after = layer_of(layer, hidden, pos, watched)
        log.append((layer, hidden.clone(), *kept, after.clone()))
        return after

    def store_prompt(layer, r, k, v):
        rows[layer, r] = k.clone(), v.clone()
        store(layer, r, k, v)

    def dense_attention(q, k, v, layer):
        out = dense(q, k, v, layer)
        steps.append((layer, *(x.clone() for x in (q, k, v, out))))
        return out
    dec._prompt_layer, dec._store_prompt, dec._dense_attention = prompt_layer, store_prompt, dense_attention
    return log, rows, steps


def attention_is(out, q, k, v, first):
    """`out` is the attention of q, whose row i sees keys 0 .. first + i, to its roundings; an output of zeros would not be."""
    o, tol, _, _ = attention64.attend(q, k, v, q.shape[2] ** -0.5, torch.arange(q.shape[0]) + first)
    attention64.check(out.view(o.shape), o, tol)
    with pytest.raises(AssertionError, match="off by"):
        attention64.check(torch.zeros_like(o), o, tol)


# Roundings of a layer's hidden state behind the attention's output: 10 (output projection, sum, norm, gate and up, silu, their
# product, down projection, sum; two more for what torch's products round inside), each by 2^-8 at most
LAYER = 10 * 2.0 ** -8


def layer_is(dec, layer, hidden, attn, after):
    """The rest of the layer in f32 from the attention's own output; from an output of zeros it would be another."""
    W, eps = dec.layers[layer], dec.shape.rms_norm_eps

    def rest(a):
        h = hidden.float() + a.reshape(hidden.shape[0], -1).float() @ W["wo"].float().t()
        y = h / torch.sqrt((h * h).mean(-1, keepdim=True) + eps) * W["ln2"].float()
        return h + (torch.nn.functional.silu(y @ W["gate"].float().t()) * (y @ W["up"].float().t())) @ W["down"].float().t()
    want = rest(attn)
    close(after, want, bound=LAYER)
    with pytest.raises(AssertionError, match="differ"):
        close(after, rest(torch.zeros_like(attn)), bound=LAYER)


@pytest.mark.gpu
@pytest.mark.parametrize("head_dim", [64, 128])
def test_every_layer_of_a_packed_prefill(head_dim):
    dec = decoder(head_dim)
    log, rows, _ = record(dec)
    lens = (400, 130)
    dec.prefill(prompts(*lens))
    assert [x[0] for x in log] == [0, 1, 2]
    for layer, hidden, q, k, v, out, after in log:
        for r, (a, b) in enumerate(((0, 400), (400, 530))):
            attention_is(out[a:b], q[a:b], k[a:b], v[a:b], 0)
            assert torch.equal(rows[layer, r][0], k[a:b]) and torch.equal(rows[layer, r][1], v[a:b])
        layer_is(dec, layer, hidden, out, after)


@pytest.mark.gpu
@pytest.mark.parametrize("chunk", [150, 97])
@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
def test_every_layer_of_a_chunked_prefill(fmt, chunk):
    """Each chunk's attention is over the rows as the cache's format holds them, and these are the rows the state gets."""
    dec = decoder(dense_cache="bf16")
    log, rows, _ = record(dec)
    dec.prefill_chunked(1, prompts(400)[0], chunk=chunk, kv_format=fmt)
    for layer in range(3):
        mine = [x for x in log if x[0] == layer]
        k, v = (stored(torch.cat([x[i] for x in mine]), fmt) for i in (3, 4))
        assert [x[2].shape[0] for x in mine] == [min(chunk, 400 - i) for i in range(0, 400, chunk)]
        for i, (_, hidden, q, _, _, out, after) in enumerate(mine):
            seen = i * chunk + q.shape[0]
            attention_is(out, q, k[:seen], v[:seen], i * chunk)
            layer_is(dec, layer, hidden, out, after)
        assert all(torch.equal(got.double(), want) for got, want in zip(rows[layer, 1], (k, v)))


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
def test_every_dense_layer_of_decode_steps_over_pages(fmt):
    """Steps behind two prompts: each dense layer's attention is over the prompt's and the steps' rows as the pages hold them."""
    dec = decoder(dense_layers=(0, 2), dense_cache=fmt)
    _, rows, steps = record(dec)
    lens = (400, 130)
    ids = dec.prefill(prompts(*lens)).argmax(-1, keepdim=True)
    for step in range(3):
        ids = dec.inference(ids, torch.tensor([[n + step] for n in lens], device="cuda"))[:, -1].argmax(-1, keepdim=True)
    dec.dense_server.check()
    for layer in (0, 2):
        mine = [x for x in steps if x[0] == layer]
        assert len(mine) == 3
        for r, n in enumerate(lens):
            k, v = rows[layer, r]
            for step, (_, q, kn, vn, out) in enumerate(mine):
                k, v = torch.cat([k, kn[r].view(1, 2, -1)]), torch.cat([v, vn[r].view(1, 2, -1)])
                attention_is(out[r], q[r].view(1, 4, -1), stored(k, fmt), stored(v, fmt), n + step)


@pytest.mark.gpu
@pytest.mark.parametrize("dense_cache", ["store", "bf16", "e4m3"])
def test_a_request_slot_is_used_again(dense_cache):
    """Another prompt, shorter or longer, in a slot that has served one: as in a decoder that never held the first."""
    a, b = decoder(dense_cache=dense_cache), decoder(dense_cache=dense_cache)
    first, second, third = prompts(700, 300, 333)
    ids = a.prefill([first, third]).argmax(-1, keepdim=True)
    for step in range(2):
        a.inference(ids, torch.tensor([[700 + step], [333 + step]], device="cuda"))
    for prompt in (second, first):
        n = prompt.numel()
        got, want = a.prefill([prompt, third]), b.prefill([prompt, third])
        assert torch.equal(got, want)
        ids, pos = want.argmax(-1, keepdim=True), torch.tensor([[n], [333]], device="cuda")
        assert torch.equal(a.inference(ids, pos), b.inference(ids, pos))


@pytest.mark.gpu
@pytest.mark.parametrize("dense_cache", ["store", "bf16"])
def test_the_shortest_and_the_longest_prompt(dense_cache):
    """69 tokens leave one outside the window; max_length - 1 leave room for one."""
    dec = decoder(dense_cache=dense_cache)
    log, _, steps = record(dec)
    ps = prompts(69, 1023)
    la = dec.prefill(ps)
    for i, p in enumerate(ps):
        close(la[i:i + 1], reference_prefill(dec, p))
    out = dec.inference(la.argmax(-1, keepdim=True), torch.tensor([[69], [1023]], device="cuda"))
    assert bool(torch.isfinite(out).all())
    dec.dense_server.check()
    dec.attention_server.window_server.check()
    _, q, k, v, got = steps[0]
    for r, (a, b) in enumerate(((0, 69), (69, 1092))):
        kk, vv = (torch.cat([x[a:b], y[r].view(1, 2, -1)]) for x, y in ((log[0][3], k), (log[0][4], v)))
        attention_is(got[r], q[r].view(1, 4, -1), kk, vv, b - a)


@pytest.mark.gpu
def test_prefill_on_two_ranks_is_the_unsharded_one():
    """Two tensor-parallel ranks as two threads on one device, partial sums meeting at a barrier, against the unsharded model."""
    import threading

    one = decoder(tp_blocks=2)
    ps = prompts(300, 71)
    want = one.prefill(ps)
    want_long = one.prefill_chunked(0, ps[0], chunk=128)
    torch.cuda.synchronize()
    meet, slot, got, errors = threading.Barrier(2, timeout=60), [None, None], [None, None], []

    def run(rank):
        def all_reduce(t):
            slot[rank] = t
            meet.wait()
            total = slot[0] + slot[1]
            meet.wait()
            t.copy_(total)
        try:
            torch.cuda.set_device(0)
            dec = decoder(tp_rank=rank, tp_world=2, all_reduce=all_reduce)
            got[rank] = dec.prefill(ps), dec.prefill_chunked(0, ps[0], chunk=128)
            torch.cuda.synchronize()
        except BaseException as e:          # noqa: BLE001 -- a failing rank must not leave the other at the barrier
            errors.append((rank, repr(e)))
            meet.abort()
    threads = [threading.Thread(target=run, args=(r,)) for r in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(timeout=90)
    assert not errors, errors
    for x, y, ref in zip(got[0], got[1], (want, want_long)):
        assert torch.equal(x, y)
        close(x, ref)


@pytest.mark.gpu
@pytest.mark.parametrize("dense_cache", ["bf16", "e4m3"])
def test_a_request_that_has_filled_its_pages(dense_cache):
    """A step behind a prompt of max_length tokens: reported, its pages as they were; the other request goes on."""
    dec = decoder(dense_cache=dense_cache)
    _, _, steps = record(dec)
    ids = dec.prefill(prompts(300, 1024)).argmax(-1, keepdim=True)
    pages = dec.dense_server.get_pages(0)[0].view(torch.uint8)
    before = pages.clone()
    dec.inference(ids, torch.tensor([[300], [1023]], device="cuda"))
    with pytest.raises(MagicPigError, match="kv_len"):
        dec.dense_server.check()
    page, slot = int(dec.dense_table[0, 300 // 64]), 300 % 64
    assert not torch.equal(pages[page, :, slot], before[page, :, slot])
    before[page, :, slot] = pages[page, :, slot]
    assert torch.equal(pages, before)
