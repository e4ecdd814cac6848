"""prompt_attention (mp_prompt_attention) against 64 bits: lengths, head groups, strides, masked infinities, rows outside the
sequences, streams and graphs; its refusals (CPU)."""
import math

import pytest
import torch

import attention64
import magicpig_amd as mp
from magicpig_amd import _lib as L


def packed(lens, H, Hkv, D, seed=0, before=0, behind=0):
    g = torch.Generator().manual_seed(seed)
    T = before + sum(lens) + behind
    q = (torch.randn((T, H, D), generator=g) * 1.5).bfloat16().cuda()
    k = (torch.randn((T, Hkv, D), generator=g) + 2 * torch.randn((1, Hkv, D), generator=g)).bfloat16().cuda()
    v = torch.randn((T, Hkv, D), generator=g).bfloat16().cuda()
    cu = torch.tensor([before] + [before + sum(lens[:i + 1]) for i in range(len(lens))], dtype=torch.int32).cuda()
    return q, k, v, cu


def compare(q, k, v, cu, out, lse, scale=None):
    scale = q.shape[2] ** -0.5 if scale is None else scale
    ends = cu.tolist()
    for a, b in zip(ends, ends[1:]):
        if b > a:
            o, t, z, zt = attention64.attend(q[a:b], k[a:b], v[a:b], scale, torch.arange(b - a))
            attention64.check(out[a:b], o, t, f"out of rows {a}..{b}")
            attention64.check(lse[a:b], z, zt, f"lse of rows {a}..{b}")


LENS = [[1], [2], [31], [32, 33], [63, 64, 65], [127, 128, 129], [0, 5, 0, 0, 7, 0], [1] * 70, [300, 1, 1000], [2049]]


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("H,Hkv", [(4, 4), (8, 2), (7, 1), (6, 2), (64, 2)])
@pytest.mark.parametrize("lens", LENS, ids=lambda x: "x".join(map(str, x[:6])))
def test_against_64_bits(lens, H, Hkv, D):
    q, k, v, cu = packed(lens, H, Hkv, D, seed=H + D)
    out, lse = mp.prompt_attention(q, k, v, cu)
    compare(q, k, v, cu, out, lse)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
def test_strided_inputs_and_scale(D):
    lens, H, Hkv = [70, 3, 200], 8, 2
    q, k, v, cu = packed(lens, H, Hkv, D, seed=5)
    qkv = torch.cat([q, k, v], dim=1)
    want = mp.prompt_attention(q, k, v, cu, scale=0.3)
    compare(q, k, v, cu, *want, scale=0.3)
    fused = mp.prompt_attention(qkv[:, :H], qkv[:, H:H + Hkv], qkv[:, H + Hkv:], cu, scale=0.3)
    heads_first = mp.prompt_attention(*(x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k, v)), cu, scale=0.3)
    for got in (fused, heads_first):
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.gpu
def test_rows_outside_the_sequences_stay():
    q, k, v, cu = packed([40, 90], 8, 2, 128, seed=6, before=3, behind=50)
    out, lse = torch.full_like(q, 7.0), torch.full((q.shape[0], 8), -3.0, device="cuda")
    mp.prompt_attention(q, k, v, cu, out=out, lse=lse)
    compare(q, k, v, cu, out, lse)
    for a, b in ((0, 3), (133, q.shape[0])):
        assert bool((out[a:b] == 7.0).all()) and bool((lse[a:b] == -3.0).all())


# few rows; more than 2^14; more than 2^17 of long sequences: workgroups of 32, 128 and 256 rows
SIZES = [([70, 3, 200], 8, 2), ([400, 3, 300], 32, 4), ([2100, 2300], 32, 8)]


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lens,H,Hkv", SIZES, ids=["32", "128", "256"])
def test_every_kernel_on_slices_outside_rows_and_nonfinite_tokens(lens, H, Hkv, D):
    q, k, v, cu = packed(lens, H, Hkv, D, seed=31, before=2, behind=3)
    ends = cu.tolist()
    v[ends[1] - 1, 0, 1] = float("inf")                    # the last token of the first sequence
    v[ends[1] - 2, Hkv - 1, D - 1] = float("nan")
    v[ends[-2] + 40, 0] = float("-inf")                    # the 41st of the last
    k[ends[-1] - 1, Hkv - 1, 0] = float("nan")
    q[0] = k[1] = v[-1] = k[-2] = float("nan")             # rows of no sequence
    qkv = torch.cat([q, k, v], dim=1)
    out, lse = torch.full_like(q, 7.0), torch.full((q.shape[0], H), -3.0, device="cuda")
    mp.prompt_attention(qkv[:, :H], qkv[:, H:H + Hkv], qkv[:, H + Hkv:], cu, out=out, lse=lse)
    compare(q, k, v, cu, out, lse)
    assert bool(torch.isfinite(out[ends[0]:ends[1] - 2]).all()) and bool(torch.isfinite(out[ends[-2]:ends[-2] + 40]).all())
    for a, b in ((0, ends[0]), (ends[-1], q.shape[0])):
        assert bool((out[a:b] == 7.0).all()) and bool((lse[a:b] == -3.0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lens,H,Hkv", SIZES, ids=["32", "128", "256"])
def test_every_kernel_on_growing_and_falling_logits(lens, H, Hkv, D):
    """Logits that climb by thousands along the keys (the running maximum has to follow again and again) and fall back."""
    q, k, v, cu = packed(lens, H, Hkv, D, seed=32)
    ramp = torch.linspace(0, 30, q.shape[0], device="cuda")[:, None, None]
    for ks in (k * ramp, k * ramp.flip(0)):
        ks = (ks + q[:, :Hkv] * ramp).bfloat16()
        compare(q, ks, v, cu, *mp.prompt_attention(q, ks, v, cu))


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_nonfinite_tokens_reach_only_rows_that_see_them(bad, D):
    q, k, v, cu = packed([150, 77], 8, 2, D, seed=7)
    v[100, 1, 5] = bad
    v[149, 0] = bad
    k[150 + 76, 0, 3] = bad
    v[150 + 70, 1, D - 1] = -bad
    v[150 + 71, 1, D - 1] = bad
    out, lse = mp.prompt_attention(q, k, v, cu)
    compare(q, k, v, cu, out, lse)
    assert bool(torch.isfinite(out[:100]).all()) and bool(torch.isfinite(out[150:220]).all())


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lens,H,Hkv", SIZES, ids=["32", "128", "256"])
def test_rows_whose_logits_are_all_minus_infinity(lens, H, Hkv, D):
    """The first keys of a sequence hold an infinity: a row that sees nothing but logits of -inf is 0 / 0, its log-sum-exp -inf;
    rows behind them have a weight of 0 there."""
    q, k, v, cu = packed(lens, H, Hkv, D, seed=38)
    for a, n in ((cu[0], 40), (cu[2] if len(lens) > 2 else cu[1], 100)):
        k[a:a + n, 0, 3] = float("inf")
        q[a:, :H // Hkv, 3] = -q[a:, :H // Hkv, 3].abs() - 0.5
    out, lse = mp.prompt_attention(q, k, v, cu)
    assert bool(torch.isnan(out[0, 0]).all()) and float(lse[0, 0]) == float("-inf")
    compare(q, k, v, cu, out, lse)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lens,H,Hkv", SIZES, ids=["32", "128", "256"])
def test_values_up_to_the_end_of_the_range(lens, H, Hkv, D):
    """v times a power of two, up to 2^120 / keys: the outputs times that power, bit for bit, while the maximum lags behind
    climbing logits."""
    q, k, v, cu = packed(lens, H, Hkv, D, seed=39)
    n = max(lens)
    ramp = torch.linspace(0, 1, q.shape[0], device="cuda")[:, None, None]
    k = (k + 0.3 * q[:, :Hkv] * ramp).bfloat16()
    v = v.clamp(-4, 4)
    big = 2.0 ** (117 - math.ceil(math.log2(n)))
    (out, lse), (far, same) = mp.prompt_attention(q, k, v, cu), mp.prompt_attention(q, k, v * big, cu)
    compare(q, k, v, cu, out, lse)
    assert bool(torch.isfinite(far).all()) and torch.equal(far.double(), out.double() * big) and torch.equal(same, lse)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lens,H,Hkv", SIZES, ids=["32", "128", "256"])
def test_logits_up_to_the_end_of_the_range(lens, H, Hkv, D):
    """|scale q . k| up to 2^24, climbing and falling: finite, within the error of f32 logits."""
    q, k, v, cu = packed(lens, H, Hkv, D, seed=41)
    ramp = torch.linspace(0.1, 1, q.shape[0], device="cuda")[:, None, None]
    for ks in ((k * ramp).bfloat16(), (k * ramp.flip(0)).bfloat16()):
        top = max(float((q[:, h].float() @ ks[:, h * Hkv // H].float().t()).abs().max()) for h in range(H))
        scale = 0.99 * 2.0 ** 24 / top
        out, lse = mp.prompt_attention(q, ks, v, cu, scale=scale)
        assert bool(torch.isfinite(out).all()) and bool(torch.isfinite(lse).all())
        compare(q, ks, v, cu, out, lse, scale=scale)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lens,H,Hkv", SIZES, ids=["32", "128", "256"])
def test_infinite_values_of_vanishing_weight(lens, H, Hkv, D):
    """A visible infinity in V whose weight is below f32's range: an infinity or NaN in its dim, nothing elsewhere."""
    q, k, v, cu = packed(lens, H, Hkv, D, seed=40)
    a, b = int(cu[-2]), int(cu[-1])
    q[a:, :H // Hkv, 0] = 8.0
    k[a:b, 0, 0] = torch.linspace(0, 800, b - a, device="cuda").bfloat16()
    v[a + 1, 0, 5], v[a + 70, 0, 6] = float("inf"), float("-inf")
    out, lse = mp.prompt_attention(q, k, v, cu)
    for dim, key in ((5, a + 1), (6, a + 70)):
        group = out[:, :H // Hkv, dim]
        assert not bool(torch.isfinite(group[key:b]).any()) and bool(torch.isfinite(group[:key]).all())
        out[key:b, :H // Hkv, dim] = 0.0
        v[key, 0, dim] = 0.0
    keep = torch.ones(D, dtype=torch.bool, device="cuda")
    keep[5] = keep[6] = False
    for i, j in zip(cu.tolist(), cu.tolist()[1:]):
        o, t, z, zt = attention64.attend(q[i:j], k[i:j], v[i:j], D ** -0.5, torch.arange(j - i))
        attention64.check(out[i:j][..., keep], o[..., keep], t[..., keep])
        attention64.check(lse[i:j], z, zt)


@pytest.mark.gpu
def test_peaked_and_flat_rows():
    """Logits of thousands next to zeros: the maximum moves far and late, weights underflow."""
    q, k, v, cu = packed([500], 4, 2, 128, seed=8)
    q[100:200] *= 100
    k[300] *= 60
    q[400:] = 0
    out, lse = mp.prompt_attention(q, k, v, cu)
    compare(q, k, v, cu, out, lse)


@pytest.mark.gpu
def test_captured_on_a_side_stream_and_replayed():
    q, k, v, cu = packed([130, 5, 61], 8, 2, 128, seed=9)
    out, lse = torch.empty_like(q), torch.empty((q.shape[0], 8), device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        mp.prompt_attention(q, k, v, cu, out=out, lse=lse)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        mp.prompt_attention(q, k, v, cu, out=out, lse=lse)
    for step in range(3):
        q2, k2, v2, cu2 = packed([100 - step, 31, 65 + step], 8, 2, 128, seed=20 + step)
        for a, b in ((q, q2), (k, k2), (v, v2), (cu, cu2)):
            a.copy_(b)
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        again = mp.prompt_attention(q, k, v, cu)
        assert torch.equal(out, again[0]) and torch.equal(lse, again[1])
        compare(q, k, v, cu, out, lse)


@pytest.mark.gpu
@pytest.mark.parametrize("H,Hkv", [(4, 2), (32, 8)])
def test_strides_beyond_2_to_the_31(H, Hkv):
    """Rows 2^20 elements apart in a buffer of more than 4 GB."""
    q, k, v, cu = packed([2000, 150], H, Hkv, 64, seed=37)
    buf = torch.empty(2150 << 20, dtype=torch.bfloat16, device="cuda")
    wide, at = [], 0
    for x in (q, k, v):
        wide.append(buf.as_strided(x.shape, (1 << 20, 64, 1), at))
        wide[-1].copy_(x)
        at += x.shape[1] * 64
    want, got = mp.prompt_attention(q, k, v, cu), mp.prompt_attention(*wide, cu)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.gpu
@pytest.mark.parametrize("n", [65, 700, 5000])
def test_many_sequences(n):
    """Every sequence is found among n, empty ones between them."""
    lens = [(7 * i) % 4 for i in range(n)]
    q, k, v, cu = packed(lens, 4, 2, 64, seed=33, before=1, behind=1)
    out, lse = mp.prompt_attention(q, k, v, cu)
    T, G = q.shape[0], 2
    seq = torch.repeat_interleave(torch.arange(n), torch.tensor(lens)).cuda()      # all sequences as one masked product
    x = torch.einsum("ihd,jhd->hij", q[1:-1].double(), k[1:-1].double().repeat_interleave(G, 1)) / 8
    i = torch.arange(T - 2, device="cuda")
    x = x.masked_fill((seq[:, None] != seq[None, :]) | (i[None, :] > i[:, None]), float("-inf"))
    p, vv = x.softmax(-1), v[1:-1].double().repeat_interleave(G, 1)
    want, mag = (torch.einsum("hij,jhd->ihd", p, y) for y in (vv, vv.abs()))
    # up to 3 keys: the bound of attention64 with logits of at most 64 products of N(0, 1.5) x N(0, 2.3)
    attention64.check(out[1:-1], want, attention64.BF16 * (want.abs() + mag) * 1.01 + 1e-4 * mag)
    attention64.check(lse[1:-1], (torch.logsumexp(x, -1) / math.log(2.0)).t(), torch.full((T - 2, 4), 1e-4, device="cuda"))


@pytest.mark.gpu
@pytest.mark.parametrize("B", [2, 63, 64, 65])
@pytest.mark.parametrize("H,Hkv", [(32, 8), (7, 1)])
def test_uneven_sequences_on_both_sides_of_a_wave(B, H, Hkv):
    """Lengths of 0 to 700 in mixed order; a lane stands for a sequence while they are at most 64."""
    lens = [(i * 389 + 650) % 701 if i % 5 != 3 else i % 2 for i in range(B)]
    q, k, v, cu = packed(lens, H, Hkv, 64, seed=B, before=1, behind=2)
    out, lse = torch.full_like(q, 7.0), torch.full((q.shape[0], H), -3.0, device="cuda")
    mp.prompt_attention(q, k, v, cu, out=out, lse=lse)
    compare(q, k, v, cu, out, lse)
    assert bool((out[0] == 7.0).all()) and bool((out[-2:] == 7.0).all()) and bool((lse[-2:] == -3.0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("H,Hkv", [(8, 2), (64, 8)])
def test_offsets_that_are_none_stay_inside(H, Hkv):
    """Offsets that fall, or lie outside: results are unspecified, memory around the outputs is not touched."""
    q, k, v, _ = packed([600], H, Hkv, 128, seed=34)
    for offsets in ([0, 500, 100, 600], [-70, 300, 2000], [600, 0], [900, 1000], [-5, -1], [0, 600, 600, 0, 600]):
        whole = torch.full((800, H, 128), 7.0, device="cuda", dtype=torch.bfloat16)
        sums = torch.full((800, H), -3.0, device="cuda")
        mp.prompt_attention(q, k, v, torch.tensor(offsets, dtype=torch.int32).cuda(), out=whole[100:700], lse=sums[100:700])
        for rows in (slice(0, 100), slice(700, 800)):
            assert bool((whole[rows] == 7.0).all()) and bool((sums[rows] == -3.0).all())


@pytest.mark.gpu
def test_gradients_are_refused():
    q, k, v, cu = packed([4], 8, 2, 128)
    q.requires_grad_()
    with pytest.raises(ValueError, match="no backward"):
        mp.prompt_attention(q, k, v, cu)
    with torch.no_grad():
        mp.prompt_attention(q, k, v, cu)


@pytest.mark.gpu
def test_forward_gradients_are_refused():
    q, k, v, cu = packed([4], 8, 2, 128)
    t = torch.ones_like(v)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(v, t)
        with pytest.raises(ValueError, match="v: .*tangent"):
            mp.prompt_attention(q, k, dual, cu)
        mp.prompt_attention(q, k, v, cu)                   # an open level alone is no reason
    with pytest.raises(ValueError, match="v: .*tangent"):
        torch.func.jvp(lambda x: mp.prompt_attention(q, k, x, cu)[0], (v,), (t,))
    for name, x in (("out", torch.empty_like(q)), ("lse", torch.empty((4, 8), device="cuda"))):
        with pytest.raises(ValueError, match=name + ": requires a gradient"):
            mp.prompt_attention(q, k, v, cu, **{name: x.requires_grad_()})


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lens,H,Hkv", SIZES, ids=["32", "128", "256"])
def test_outputs_beside_inputs_and_over_the_queries(lens, H, Hkv, D):
    q, k, v, cu = packed(lens, H, Hkv, D, seed=42)
    want = mp.prompt_attention(q, k, v, cu)
    T = q.shape[0]
    room = torch.zeros(T * (2 * H + 2 * Hkv) * D, dtype=torch.bfloat16, device="cuda")       # all four, one behind the other
    qq, oo, kk, vv = (x.view(T, -1, D) for x in room.split([T * H * D, T * H * D, T * Hkv * D, T * Hkv * D]))
    for x, y in ((qq, q), (kk, k), (vv, v)):
        x.copy_(y)
    got = mp.prompt_attention(qq, kk, vv, cu, out=oo)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    got = mp.prompt_attention(qq, kk, vv, cu, out=qq)
    assert got[0] is qq and torch.equal(qq, want[0]) and torch.equal(got[1], want[1])
    with pytest.raises(mp.MagicPigError, match="overlap"):
        mp.prompt_attention(oo, kk, vv, cu, out=room[8:T * H * D + 8].view(T, H, D))


@pytest.mark.gpu
def test_one_token_in_one_fused_row():
    """q, k, v and the output side by side in one row."""
    q, k, v, cu = packed([1], 8, 2, 128, seed=43)
    row = torch.cat([q, k, v, torch.zeros_like(q)], dim=1)
    out, _ = mp.prompt_attention(row[:, :8], row[:, 8:10], row[:, 10:12], cu, out=row[:, 12:])
    assert torch.equal(out, v.repeat_interleave(4, 1)) and torch.equal(row[:, 12:], out)


@pytest.mark.gpu
def test_empty_inputs():
    q, k, v, cu = packed([0, 0], 8, 2, 128)
    out, lse = mp.prompt_attention(q, k, v, cu)
    assert out.shape == (0, 8, 128) and lse.shape == (0, 8)


@pytest.mark.gpu
def test_refusals_of_shapes_and_devices():
    q, k, v, cu = packed([4], 8, 2, 128)
    for args, word in (((q, k[:, :, :64], v, cu), "k: expected shape"), ((q, k[:3], v, cu), "tokens"), ((q, k, v[:, :1], cu), "v: expected"),
                       ((q, k, v, cu.cpu()), "cu_seqlens: on cpu"), ((q, k, v, cu[:1]), "cu_seqlens"),
                       ((q[:, :, ::2], k[:, :, ::2], v[:, :, ::2], cu), "contiguous")):
        with pytest.raises(ValueError, match=word):
            mp.prompt_attention(*args)
    with pytest.raises(TypeError, match="cu_seqlens"):
        mp.prompt_attention(q, k, v, cu.long())


# ---------------------------------------------------------------- refusals: nothing reaches the GPU
GOOD = dict(q=1 << 20, qt=1024, qh=128, k=1 << 20, kt=256, kh=128, v=1 << 20, vt=256, vh=128, cu=1 << 20, seqs=2, tokens=10,
            H=8, Hkv=2, D=128, scale=0.1, out=1 << 20, lse=1 << 20, stream=None)


@pytest.mark.parametrize("change,code", [
    (dict(D=96), 5), (dict(D=256), 5), (dict(H=7), 1), (dict(H=1), 1), (dict(Hkv=0), 1), (dict(seqs=0), 1), (dict(tokens=-1), 1),
    (dict(scale=0.0), 1), (dict(scale=-1.0), 1), (dict(scale=float("nan")), 1), (dict(scale=float("inf")), 1),
    (dict(q=None), 1), (dict(k=None), 1), (dict(v=None), 1), (dict(cu=None), 1), (dict(out=None), 1),
    (dict(q=(1 << 20) + 2), 1), (dict(k=(1 << 20) + 8), 1), (dict(v=(1 << 20) + 4), 1), (dict(out=(1 << 20) + 8), 1),
    (dict(qt=1020), 1), (dict(kh=12), 1), (dict(vt=-256), 1), (dict(vt=1 << 23), 1), (dict(tokens=1 << 29), 5),
    (dict(seqs=(1 << 31) - 1), 5), (dict(tokens=1 << 27, H=64), 5)])
def test_refusals_of_the_c_entry(change, code):
    a = {**GOOD, **change}
    assert L.lib().mp_prompt_attention(*(a[n] for n in GOOD)) == code
    assert b"mp_prompt_attention" in L.lib().mp_last_error()


@pytest.mark.parametrize("scale", [2.4e38, 3.4e38])
def test_a_scale_that_is_infinite_in_base_2_is_refused(scale):
    far = dict(q=1 << 40, k=2 << 40, v=3 << 40, out=4 << 40, lse=5 << 40)
    assert L.lib().mp_prompt_attention(*({**GOOD, **far, "scale": scale, "tokens": 0}[n] for n in GOOD)) == 1
    assert b"scale" in L.lib().mp_last_error()


BASE, T, ROW = 1 << 24, 10, 128 * 2          # 10 tokens; bytes of a head's row


@pytest.mark.parametrize("change", [
    dict(out=BASE, k=BASE + 8 * ROW), dict(out=BASE, k=BASE + T * 8 * ROW - 16), dict(out=BASE, v=BASE - T * 2 * ROW + 16),
    dict(out=BASE, q=BASE + 16), dict(out=BASE, q=BASE, qt=2048), dict(out=BASE, q=BASE, qh=T * 128, qt=128), dict(out=BASE, q=BASE - T * 8 * ROW + 16),
    dict(out=BASE, lse=BASE + T * 8 * ROW - 4), dict(out=BASE, lse=BASE - 4), dict(lse=BASE, q=BASE), dict(lse=BASE, k=BASE - T * 2 * ROW + 16),
    dict(lse=BASE, v=BASE + T * 8 * 4 - 16), dict(out=BASE, k=BASE - 9 * 8192 * 2, kt=8192), dict(out=1 << 45, v=1 << 44, vh=1 << 43, vt=1 << 20),
    dict(out=BASE, k=BASE, kt=0, kh=0), dict(out=BASE, k=BASE - (1 << 20), kh=(1 << 62) + (1 << 61), kt=(1 << 23) - 8)])
def test_outputs_over_inputs_are_refused(change):
    far = dict(q=1 << 40, k=2 << 40, v=3 << 40, out=4 << 40, lse=5 << 40)
    a = {**GOOD, "tokens": T, **far, **change}
    assert L.lib().mp_prompt_attention(*(a[n] for n in GOOD)) == 1
    assert b"overlap" in L.lib().mp_last_error()


def test_refusals_of_the_python_entry():
    x = torch.zeros((4, 8, 128), dtype=torch.bfloat16)
    kv = torch.zeros((4, 2, 128), dtype=torch.bfloat16)
    cu = torch.tensor([0, 4], dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        mp.prompt_attention(x, kv, kv, cu)
    with pytest.raises(TypeError, match="dtype"):
        mp.prompt_attention(x.float(), kv, kv, cu)
    with pytest.raises(ValueError, match="q:"):
        mp.prompt_attention(x[0], kv, kv, cu)
