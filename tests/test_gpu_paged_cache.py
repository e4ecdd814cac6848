"""PagedKVCache (mp_paged_*): rows written and read back (bf16, e4m3), attention over pages against 64 bits, bad pages and
lengths, streams, graphs and shared pages; refusals (CPU)."""
import ctypes as C

import pytest
import torch

import attention64
import magicpig_amd as mp
from magicpig_amd import _lib as L


def stored(x, fmt):
    """What rows x (bf16) come back as, in 64 bits: nearest of the 3-bit numbers with exponents from -6 up to 448, ties to
    even, of x over the least power of two that brings the row's largest finite magnitude to at most 448."""
    if fmt == "bf16":
        return x.double()
    y = x.double().cpu()
    top = torch.where(torch.isfinite(y), y.abs(), 0.0).amax(-1, keepdim=True)
    e = torch.full_like(top, -126.0)
    for _ in range(300):
        e = torch.where(top > 448.0 * torch.exp2(e), e + 1, e)
    z = y * torch.exp2(-e)
    unit = torch.exp2(torch.frexp(z.abs().nan_to_num(1.0, 1.0, 1.0).clamp(min=2.0 ** -6))[1].double() - 4)
    z = torch.round(z / unit) * unit * torch.exp2(e)
    return torch.where(torch.isfinite(y), z, float("nan")).to(x.device)


class Setup:
    """Requests of (new, kv) tokens over shuffled pages, spare pages among them."""

    def __init__(self, pairs, page, H, Hkv, D, fmt, seed=0, layers=1, before=0, behind=0, spare=3, layer=0):
        self.pairs, self.page, self.H, self.Hkv, self.D, self.fmt, self.layer = pairs, page, H, Hkv, D, fmt, layer
        g = torch.Generator().manual_seed(seed)
        self.g = g
        need = [-(-kv // page) for _, kv in pairs]
        P = max(max(need), 1)
        order = torch.randperm(sum(need) + spare, generator=g)
        self.table = torch.full((len(pairs), P), -1, dtype=torch.int32)      # entries behind a request's pages: never used
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = order[at:at + n]
            at += n
        self.table = self.table.cuda()
        news = [n for n, _ in pairs]
        self.ends = [before + sum(news[:i]) for i in range(len(news) + 1)]
        self.T = self.ends[-1] + behind
        self.cu = torch.tensor(self.ends, dtype=torch.int32).cuda()
        self.kv_len = torch.tensor([c for _, c in pairs], dtype=torch.int32).cuda()
        self.cache = mp.PagedKVCache()
        self.cache.alloc(layers, H, Hkv, D, sum(need) + spare, page, kv_format=fmt)
        mean = 2 * torch.randn((1, Hkv, D), generator=g)
        self.k = [(torch.randn((kv, Hkv, D), generator=g) + mean).bfloat16().cuda() for _, kv in pairs]
        self.v = [torch.randn((kv, Hkv, D), generator=g).bfloat16().cuda() for _, kv in pairs]
        self.q = (torch.randn((self.T, H, D), generator=g) * 1.5).bfloat16().cuda()

    def fill(self):
        kv = [c for _, c in self.pairs]
        cu = torch.tensor([sum(kv[:i]) for i in range(len(kv) + 1)], dtype=torch.int32).cuda()
        self.cache.append(self.layer, torch.cat(self.k), torch.cat(self.v), cu, self.table, self.kv_len)
        return self

    def attend(self, **kw):
        return self.cache.attention(self.layer, self.q, self.cu, self.table, self.kv_len, **kw)

    def compare(self, out, lse, scale=None):
        scale = self.D ** -0.5 if scale is None else scale
        for b, (n, kv) in enumerate(self.pairs):
            rows = slice(self.ends[b], self.ends[b + 1])
            if n:
                o, t, z, zt = attention64.attend(self.q[rows], stored(self.k[b], self.fmt), stored(self.v[b], self.fmt), scale,
                                                 torch.arange(n) + kv - n)
                attention64.check(out[rows], o, t, f"out of request {b}")
                attention64.check(lse[rows], z, zt, f"lse of request {b}")
        self.cache.check()


# ---------------------------------------------------------------- rows in and out
@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("page,pairs,Hkv", [
    (1, [(1, 1), (3, 9)], 1), (8, [(5, 5), (0, 4), (1, 30), (16, 16)], 2), (64, [(1, 65)] * 20, 3),
    (16, [(77, 200), (130, 130)], 8), (256, [(300, 1000), (2, 2)], 2)])
def test_append_then_read(page, pairs, Hkv, D, fmt):
    s = Setup(pairs, page, Hkv, Hkv, D, fmt, seed=page, layers=2, layer=1, before=2, behind=5)
    k, v = torch.randn((2, s.T, Hkv, D), generator=s.g).bfloat16().cuda() * torch.exp2(
        torch.randint(-30, 30, (2, s.T, Hkv, 1), generator=s.g).float()).bfloat16().cuda()
    pages, scales = (x.view(torch.uint8) if x is not None else None for x in s.cache.get_pages(1))
    pages.fill_(0x5a)
    s.cache.append(1, k, v, s.cu, s.table, s.kv_len)
    ko, vo = torch.full_like(k, 9.0), torch.full_like(v, 9.0)
    s.cache.read(1, s.T, s.cu, s.table, s.kv_len, k=ko, v=vo)
    s.cache.check()
    inside = slice(s.ends[0], s.ends[-1])
    for got, x in ((ko, k), (vo, v)):
        assert torch.equal(got[inside].double(), stored(x[inside], fmt))
        assert bool((got[:s.ends[0]] == 9.0).all()) and bool((got[s.ends[-1]:] == 9.0).all())
    # nothing else changed: the places of new rows, all other bytes as they were
    mine = torch.zeros((s.cache.num_pages, page), dtype=torch.bool)
    for b, (n, kv) in enumerate(pairs):
        for pos in range(kv - n, kv):
            mine[int(s.table[b, pos // page]), pos % page] = True
    rest = pages.permute(0, 2, 1, 3, 4)[~mine.cuda()]
    assert bool((rest == 0x5a).all())
    assert int(s.cache.get_pages(0)[0].view(torch.uint8).max()) == 0
    if scales is not None:
        assert int(scales.permute(0, 2, 1, 3)[~mine.cuda()].max()) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
def test_quantised_corner_rows(D):
    """Rows of zeros, of one value, at the borders 448 * 2^e, of subnormals, of the largest numbers, with infinities and NaN."""
    big = torch.finfo(torch.bfloat16).max
    firsts = [0.0, 1.0, 448.0, 450.0, 446.0, 1.75, 1.7578125, 2.0 ** -126, 2.0 ** -133, 3 * 2.0 ** -133, big, 2.0 ** 100,
              float("inf"), float("nan"), -448.0, 7 * 2.0 ** -120]
    g = torch.Generator().manual_seed(3)
    k = torch.rand((len(firsts), 1, D), generator=g) * 2 - 1
    for i, x in enumerate(firsts):
        m = abs(x) if x == x and abs(x) != float("inf") else 5.0
        k[i] *= min(m, big)
        k[i, 0, i % D] = x
        k[i, 0, (i + 7) % D] = m * 2.0 ** -9
        k[i, 0, (i + 9) % D] = -m * 2.0 ** -17
    k = k.bfloat16().cuda()
    s = Setup([(len(firsts), len(firsts))], 8, 1, 1, D, "e4m3")
    s.cache.append(0, k, -k, s.cu, s.table, s.kv_len)
    ko, vo = s.cache.read(0, len(firsts), s.cu, s.table, s.kv_len)
    # below bf16's normal range the product with 2^e is rounded to bf16 once more
    want = stored(k, "e4m3").to(torch.float32).bfloat16()
    for got, w in ((ko, want), (vo, -want)):
        assert torch.equal(torch.isnan(got), torch.isnan(w))
        assert torch.equal(got[~torch.isnan(w)], w[~torch.isnan(w)])


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
def test_strided_rows_and_rows_without_a_place(fmt):
    s = Setup([(4, 4), (5, 2), (2, 0), (3, 40)], 16, 4, 2, 128, fmt, seed=4)
    qkv = torch.randn((s.T, 8, 128), generator=s.g).bfloat16().cuda()
    k, v = qkv[:, 4:6], qkv[:, 6:]
    s.cache.append(0, k, v, s.cu, s.table, s.kv_len)
    ko, vo = torch.full((2, s.T, 2, 128), 9.0, device="cuda", dtype=torch.bfloat16)
    s.cache.read(0, s.T, s.cu, s.table, s.kv_len, k=ko, v=vo)
    s.cache.check()
    lost = torch.zeros(s.T, dtype=torch.bool)
    lost[4:7] = True                     # request 1: 5 new rows, 2 positions; request 2: none
    lost[9:11] = True
    for got, x in ((ko, k), (vo, v)):
        assert torch.equal(got[~lost].double(), stored(x[~lost], fmt))
        assert bool((got[lost] == 9.0).all())


# ---------------------------------------------------------------- attention
CASES = [
    (64, [(1, 1)]), (64, [(1, 64), (1, 65), (1, 63), (1, 2)]), (1, [(1, 33), (2, 90)]), (16, [(1, 5000)]),
    (32, [(1, 700), (4, 4), (0, 100), (7, 1000), (1, 0), (3, 2)]), (128, [(33, 33), (64, 500)]), (256, [(130, 130), (1, 3000)]),
    (64, [(300, 1500)]), (8, [(1, 40 * i + 1) for i in range(40)]), (64, [(700, 700), (1, 20)]),
]


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
@pytest.mark.parametrize("H,Hkv,D", [(8, 2, 128), (8, 1, 64), (3, 3, 128), (14, 2, 64), (64, 1, 128)])
@pytest.mark.parametrize("page,pairs", CASES, ids=[f"page{p}-" + "-".join(f"{n}of{c}" for n, c in r[:3]) for p, r in CASES])
def test_attention_against_64_bits(page, pairs, H, Hkv, D, fmt):
    s = Setup(pairs, page, H, Hkv, D, fmt, seed=H).fill()
    s.compare(*s.attend())


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("pairs,H,Hkv", [
    ([(40, 20000)], 32, 8), ([(300, 6000), (1, 9), (77, 5000)], 16, 4), ([(1500, 1500)], 32, 8), ([(5000, 5000), (300, 200)], 32, 8)])
def test_workgroups_of_many_rows_whole_and_in_parts(pairs, H, Hkv, D, fmt):
    s = Setup(pairs, 64, H, Hkv, D, fmt, seed=21).fill()
    s.compare(*s.attend())


def workspace(s):
    need = C.c_int64()
    L.check(L.lib().mp_paged_workspace(s.cache._h, len(s.pairs), s.T, s.table.shape[1], C.byref(need)))
    return need.value


# 128 rows a workgroup: tables of at most 512 positions and more rows than the kernel for few of them takes; 256 at head_dim 128
# and 2^16 rows; rows enough to fill the chip behind longer tables
UNCUT = [([(300, 500), (17, 512), (0, 40), (90, 90), (257, 300), (60, 20)], 32, 8), ([(500, 512), (1, 3), (511, 511), (400, 100)] * 2, 32, 8),
         ([(3000, 3500), (2500, 2500), (0, 9), (2700, 2900), (1, 700)], 32, 8)]


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("pairs,H,Hkv", UNCUT, ids=["short tables", "short tables, most rows", "a full chip"])
def test_many_rows_whose_keys_are_not_cut(pairs, H, Hkv, D, fmt):
    """A workgroup finds its tile among the requests' slots, from the last one on."""
    s = Setup(pairs, 32, H, Hkv, D, fmt, seed=27, before=3, behind=70).fill()
    assert workspace(s) == 0
    out, lse = torch.full_like(s.q, 7.0), torch.full((s.T, H), -3.0, device="cuda")
    s.attend(out=out, lse=lse)
    s.compare(out, lse)
    for rows in (slice(0, 3), slice(s.ends[-1], s.T)):
        assert bool((out[rows] == 7.0).all()) and bool((lse[rows] == -3.0).all())


@pytest.mark.gpu
def test_uncut_keys_and_offsets_that_are_none():
    pairs, H, Hkv = UNCUT[0]
    s = Setup(pairs, 32, H, Hkv, 128, "bf16", seed=28).fill()
    T = s.T
    for offsets in ([0, T, 1, 2, 3, 4, 5], [-9, T // 2, T + 70, 0, T, T, T], [T, 0, 0, T, 0, T, 0]):
        cu = torch.tensor(offsets, dtype=torch.int32).cuda()
        whole, sums = torch.full((T + 60, H, 128), 7.0, device="cuda", dtype=torch.bfloat16), torch.full((T + 60, H), -3.0, device="cuda")
        s.cache.attention(0, s.q, cu, s.table, s.kv_len.clamp(max=500), out=whole[30:T + 30], lse=sums[30:T + 30])
        for x, value in ((whole, 7.0), (sums, -3.0)):
            assert bool((x[:30] == value).all()) and bool((x[T + 30:] == value).all())


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
@pytest.mark.parametrize("pairs,H,Hkv", [([(30, 100), (1, 600)], 8, 2), ([(300, 4000), (1, 600)], 32, 8), ([(2100, 2300), (1, 600)], 32, 8)],
                         ids=["few rows", "many rows", "most rows"])
def test_nonfinite_values_in_every_kernel(pairs, H, Hkv, fmt):
    s = Setup(pairs, 16, H, Hkv, 128, fmt, seed=22)
    s.v[0][-1, 0, 3] = float("inf")
    s.v[0][-2, 1, 4] = float("nan")
    s.v[0][-20, 0, 5] = float("-inf")
    s.v[1][-1, 1] = float("-inf")
    s.k[0][-3, Hkv - 1, 7] = float("nan")
    s.fill()
    pages, scales = s.cache.get_pages(0)
    for b, (n, kv) in enumerate(pairs):            # what lies behind a request's end: all bits set, NaN in either format
        place = (int(s.table[b, (kv - 1) // 16]), slice(None), slice((kv - 1) % 16 + 1, None))
        pages.view(torch.uint8)[place] = 255
        if scales is not None:
            scales[place] = 255
    s.compare(*s.attend())


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("pairs,H,Hkv", [
    ([(1, 9000), (3, 70)], 8, 2), ([(33, 600), (2, 0), (5, 3)], 8, 2), ([(300, 4000), (800, 750)], 8, 8), ([(400, 460), (400, 90)], 32, 8),
    ([(2100, 2300), (500, 40)], 32, 8)], ids=["step in parts", "step", "parts, a row that sees nothing", "128", "256"])
def test_rows_whose_logits_are_all_minus_infinity(pairs, H, Hkv, D):
    """Every key of a request, or its first 64, hold an infinity that makes all logits of some rows -inf: 0 / 0 there, log-sum-exp
    -inf; 0 and -inf where a row sees no key at all."""
    s = Setup(pairs, 16, H, Hkv, D, "bf16", seed=24)
    s.k[0][:, 0, 3] = float("inf")
    s.k[-1][:64, 0, 3] = float("inf")
    s.q[:, :H // Hkv, 3] = -s.q[:, :H // Hkv, 3].abs() - 0.5
    s.fill()
    out, lse = s.attend()
    assert bool(torch.isnan(out[0, 0]).all()) and float(lse[0, 0]) == float("-inf")
    s.compare(out, lse)


@pytest.mark.gpu
@pytest.mark.parametrize("pairs,H,Hkv", [([(1, 9000), (5, 700)], 8, 2), ([(300, 4000), (1, 600)], 32, 8), ([(2100, 2300), (1, 600)], 32, 8)],
                         ids=["few rows", "many rows", "most rows"])
def test_infinite_values_of_vanishing_weight(pairs, H, Hkv):
    """A visible infinity in V whose weight is below f32's range, in this part of the keys or another: an infinity or NaN in its
    dim, nothing elsewhere; the largest values that are sure to stay finite beside it."""
    s = Setup(pairs, 16, H, Hkv, 128, "bf16", seed=25)
    s.q[:, :H // Hkv, 0] = 8.0
    s.k[0][:, 0, 0] = torch.linspace(0, 1600, pairs[0][1], device="cuda").bfloat16()
    big = 2.0 ** 103
    s.v[0][:, 1:, :] = s.v[0][:, 1:, :].clamp(-4, 4) * big              # 2^105 x 2^14 keys
    s.v[0][1, 0, 5] = float("inf")
    s.fill()
    out, lse = s.attend()
    mine = out[s.ends[0]:s.ends[1], :H // Hkv, 5]
    assert not bool(torch.isfinite(mine).any())
    out[s.ends[0]:s.ends[1], :H // Hkv, 5] = 0.0
    s.v[0][:, 0, 5] = 0.0
    s.compare(out, lse)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt,layers", [("bf16", 1), ("e4m3", 3)])
def test_more_pages_than_the_memory_holds(fmt, layers):
    """The allocation fails, gives back what it had, and leaves nothing behind for the calls after it."""
    cache = mp.PagedKVCache()
    torch.cuda.synchronize()
    free = torch.cuda.mem_get_info()[0]
    rows = int(0.4 * torch.cuda.mem_get_info()[1] / 256) if layers > 1 else (1 << 32) // 2       # the third layer, or the first, does not fit
    with pytest.raises(mp.MagicPigError, match="MP_ERR_NOMEM"):
        cache.alloc(layers, 8, 1, 128, rows // 4096, 4096, kv_format=fmt)
    assert torch.equal(torch.arange(5, device="cuda") + 1, torch.arange(1, 6, device="cuda"))
    assert torch.cuda.mem_get_info()[0] > free - (1 << 30)
    with pytest.raises(mp.MagicPigError, match="not allocated"):
        L.check(L.lib().mp_paged_check(cache._h, None))
    cache.alloc(1, 8, 1, 128, 4, 64, kv_format=fmt)
    k = torch.randn((3, 1, 128), device="cuda").bfloat16()
    cu, table, n = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([0, 3], [[2]], [3]))
    cache.append(0, k, k, cu, table, n)
    assert torch.equal(cache.read(0, 3, cu, table, n)[0].double(), stored(k, fmt))
    cache.check()


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
def test_pages_beyond_4_gigabytes(fmt):
    """Requests whose pages lie at the end of a pool of more than 2^32 bytes and 2^31 elements."""
    s = Setup([(3, 700), (200, 900)], 64, 8, 4, 128, fmt, seed=23, spare=44000 if fmt == "bf16" else 90000)
    used = (s.table >= 0)
    s.table[used] = (s.cache.num_pages - 1 - torch.arange(int(used.sum()), device="cuda")).int()
    assert s.cache.footprint()["pages"] > (1 << 32) + (1 << 30)
    s.fill()
    s.compare(*s.attend())
    k, v = s.cache.read(0, s.T, s.cu, s.table, s.kv_len)
    for got, x in ((k, s.k), (v, s.v)):
        assert torch.equal(got.double(), stored(torch.cat([x[0][-3:], x[1][-200:]]), fmt))


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
def test_long_cache_in_many_parts(fmt):
    s = Setup([(1, 40000), (2, 17), (1, 9000)], 64, 8, 2, 128, fmt, seed=11).fill()
    s.compare(*s.attend(scale=0.2), scale=0.2)


@pytest.mark.gpu
def test_rows_outside_the_requests_stay_and_results_repeat():
    s = Setup([(3, 900), (40, 400)], 32, 8, 2, 128, "bf16", seed=12, before=4, behind=9).fill()
    out, lse = torch.full_like(s.q, 7.0), torch.full((s.T, 8), -3.0, device="cuda")
    s.attend(out=out, lse=lse)
    s.compare(out, lse)
    for rows in (slice(0, 4), slice(s.ends[-1], s.T)):
        assert bool((out[rows] == 7.0).all()) and bool((lse[rows] == -3.0).all())
    inside = slice(4, s.ends[-1])
    for _ in range(3):
        o, z = s.attend()
        assert torch.equal(o[inside], out[inside]) and torch.equal(z[inside], lse[inside])


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
@pytest.mark.parametrize("pairs", [[(30, 100)], [(1, 100), (2, 3000)]])
def test_nonfinite_tokens_reach_only_rows_that_see_them(pairs, bad):
    s = Setup(pairs, 16, 8, 2, 128, "bf16", seed=13)
    s.v[0][99, 0, 3] = bad
    s.v[-1][len(s.v[-1]) - 1, 1, 5] = -bad
    s.k[-1][len(s.k[-1]) - 1, 0, 6] = bad
    s.fill()
    pages = s.cache.get_pages(0)[0]
    for b, (n, kv) in enumerate(pairs):                    # and what lies behind a request's end in its last page
        pages[int(s.table[b, (kv - 1) // 16]), :, (kv - 1) % 16 + 1:] = float("nan")
    s.compare(*s.attend())


@pytest.mark.gpu
@pytest.mark.parametrize("H,Hkv,B", [(8, 1, 300), (4, 2, 1100), (8, 4, 5000)])
def test_many_requests(H, Hkv, B):
    """One new token or none of each of B short requests: whole, and (few heads) with the keys cut."""
    g = torch.Generator().manual_seed(35)
    D, page, most = 64, 4, 12
    kv = torch.randint(1, most + 1, (B,), generator=g)
    new = (torch.arange(B) % 5 != 2).long()
    rows = new.nonzero().flatten().cuda()
    cu = torch.cat([torch.zeros(1, dtype=torch.long), new.cumsum(0)]).int().cuda()
    table = torch.randperm(B * 3, generator=g).int().view(B, 3).cuda()
    k, v = ((torch.randn((B, most, Hkv, D), generator=g)).bfloat16().cuda() for _ in range(2))
    q = torch.randn((int(new.sum()), H, D), generator=g).bfloat16().cuda()
    cache = mp.PagedKVCache()
    cache.alloc(1, H, Hkv, D, B * 3, page)
    live = torch.arange(most)[None, :] < kv[:, None]
    cache.append(0, k[live.cuda()], v[live.cuda()], torch.cat([torch.zeros(1, dtype=torch.long), kv.cumsum(0)]).int().cuda(), table, kv.int().cuda())
    out, lse = cache.attention(0, q, cu, table, kv.int().cuda())
    cache.check()
    x = torch.einsum("bhd,bjhd->bhj", q.double(), k[rows].double().repeat_interleave(H // Hkv, 2)) / 8
    x = x.masked_fill(~live.cuda()[rows][:, None, :], float("-inf"))
    vv = v[rows].double().repeat_interleave(H // Hkv, 2)
    want, mag = (torch.einsum("bhj,bjhd->bhd", x.softmax(-1), y) for y in (vv, vv.abs()))
    attention64.check(out, want, attention64.BF16 * (want.abs() + mag) * 1.01 + 1e-4 * mag)
    attention64.check(lse, torch.logsumexp(x, -1) / torch.log(torch.tensor(2.0, dtype=torch.float64)), torch.full_like(lse, 1e-4).double())


@pytest.mark.gpu
@pytest.mark.parametrize("pairs", [[(3, 900), (2, 50)], [(400, 900), (2, 50)]])
def test_offsets_that_are_none_stay_inside(pairs):
    """Offsets that fall, or lie outside: results are unspecified, other memory is not touched."""
    s = Setup(pairs, 32, 16, 4, 128, "bf16", seed=36).fill()
    T = s.T
    for offsets in ([0, T, 1], [-9, T // 2, T + 70], [T, 0, 0], [T + 1, T + 5, T + 9]):
        cu = torch.tensor(offsets, dtype=torch.int32).cuda()
        whole, sums = torch.full((T + 60, 16, 128), 7.0, device="cuda", dtype=torch.bfloat16), torch.full((T + 60, 16), -3.0, device="cuda")
        s.cache.attention(0, s.q, cu, s.table, s.kv_len, out=whole[30:T + 30], lse=sums[30:T + 30])
        ko, vo = (torch.full((T + 60, 4, 128), 7.0, device="cuda", dtype=torch.bfloat16) for _ in range(2))
        s.cache.append(0, ko[30:T + 30], vo[30:T + 30], cu, s.table, s.kv_len)
        s.cache.read(0, T, cu, s.table, s.kv_len, k=ko[30:T + 30], v=vo[30:T + 30])
        for x, value in ((whole, 7.0), (sums, -3.0), (ko, 7.0), (vo, 7.0)):
            assert bool((x[:30] == value).all()) and bool((x[T + 30:] == value).all())


@pytest.mark.gpu
def test_shared_pages():
    """Two requests whose first 128 positions are the same pages."""
    s = Setup([(3, 200), (5, 300)], 32, 8, 2, 128, "e4m3", seed=14)
    s.table[1, :4] = s.table[0, :4]
    s.k[1][:128], s.v[1][:128] = s.k[0][:128], s.v[0][:128]
    s.fill()
    s.compare(*s.attend())


@pytest.mark.gpu
def test_step_captured_and_replayed_with_growing_lengths():
    """append + attention of one token a request in one graph; lengths and pages change between replays; a second graph of
    the same cache and eager calls in between."""
    pairs = [(1, 130), (1, 3), (1, 1000), (1, 0)]
    s = Setup(pairs, 64, 8, 2, 128, "e4m3", seed=15, spare=20)
    s.table = torch.cat([s.table, torch.full((4, 40 - s.table.shape[1]), -1, dtype=torch.int32, device="cuda")], 1)
    s.fill()
    kn, vn = (torch.zeros((4, 2, 128), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    outs = [torch.empty_like(s.q) for _ in range(2)]
    lses = [torch.empty((4, 8), device="cuda") for _ in range(2)]

    def step(i):
        s.cache.append(0, kn, vn, s.cu, s.table, s.kv_len)
        s.attend(out=outs[i], lse=lses[i])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        s.attend()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs = []
    for i in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[i]):
            step(i)
    free = [p for p in range(s.cache.num_pages) if p not in set(s.table[s.table >= 0].tolist())]
    for it in range(6):
        s.kv_len[:3] += 1                                   # (request 3 stays inactive)
        s.pairs = [(1, c + 1) for _, c in s.pairs[:3]] + [(1, 0)]
        for b in range(3):
            c = s.pairs[b][1]
            if (c - 1) % 64 == 0:
                s.table[b, (c - 1) // 64] = free.pop()
            x = torch.randn((2, 2, 128), generator=s.g).bfloat16().cuda()
            kn[b], vn[b] = x
            s.k[b], s.v[b] = torch.cat([s.k[b], x[:1]]), torch.cat([s.v[b], x[1:]])
        graphs[it % 2].replay()
        torch.cuda.synchronize()
        s.compare(outs[it % 2], lses[it % 2])
        o, z = s.attend()
        assert torch.equal(o, outs[it % 2]) and torch.equal(z, lses[it % 2])


@pytest.mark.gpu
def test_side_stream():
    s = Setup([(1, 2000), (3, 50)], 64, 8, 2, 64, "bf16", seed=16)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        s.fill()
        out, lse = s.attend()
    side.synchronize()
    s.compare(out, lse)


@pytest.mark.gpu
def test_bad_pages_and_lengths_are_reported():
    s = Setup([(1, 100), (2, 90)], 16, 8, 2, 128, "bf16", seed=17).fill()
    s.cache.check()
    want = s.attend()
    for table, kv_len in ((s.cache.num_pages, None), (-5, None), (None, 16 * s.table.shape[1] + 1), (None, -1)):
        t, n = s.table.clone(), s.kv_len.clone()
        if table is not None:
            t[0, 2] = table
        else:
            n[0] = kv_len
        out, _ = s.cache.attention(0, s.q, s.cu, t, n)
        with pytest.raises(mp.MagicPigError, match="MP_ERR_DATA"):
            s.cache.check()
        assert torch.equal(out[1:], want[0][1:])                       # the other request is not concerned
        t[0] = table if table is not None else t[0]
        s.cache.append(0, *(torch.cat([x[0][-1:], x[1][-2:]]) for x in (s.k, s.v)), s.cu, t, n)    # (request 1 as it is)
        s.cache.read(0, 3, s.cu, t, n)
        with pytest.raises(mp.MagicPigError, match="MP_ERR_DATA"):
            s.cache.check()
    s.cache.check()


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("more", [0, 300], ids=["few requests", "many requests"])
def test_rows_past_the_table_are_skipped(more, D, fmt):
    """A request that fills its table, and lengths that the table cannot hold: no byte of the pages changes, read leaves its
    outputs, and the next calls are as before.  Its last page is also the first of another request."""
    s = Setup([(0, 112), (2, 90)] + [(0, 1)] * more, 16, 4, 2, D, fmt, seed=18)
    s.table[1, 0] = s.table[0, 6]
    s.k[1][:16], s.v[1][:16] = s.k[0][96:], s.v[0][96:]
    s.fill()
    whole = [x.view(torch.uint8).clone() for x in s.cache.get_pages(0) if x is not None]
    for new, length in ((1, 113), (5, 115), (3, 113), (16, 112 + 16), (1, (1 << 31) - 1), (2, -1), (1, -(1 << 31))):
        kv_len = s.kv_len.clone()
        kv_len[0] = length
        cu = torch.tensor([0] + [new] + [new + 2] * (more + 1), dtype=torch.int32).cuda()
        junk = torch.full((new, 2, D), 3.0, dtype=torch.bfloat16, device="cuda")
        s.cache.append(0, torch.cat([junk, s.k[1][-2:]]), torch.cat([junk, s.v[1][-2:]]), cu, s.table, kv_len)    # (request 1 as it is)
        for now, then in zip((x for x in s.cache.get_pages(0) if x is not None), whole):
            assert torch.equal(now.view(torch.uint8), then), f"{new} rows, kv_len {length}"
        with pytest.raises(mp.MagicPigError, match="MP_ERR_DATA.*kv_len"):
            s.cache.check()
        ko, vo = (torch.full((new + 2, 2, D), 9.0, dtype=torch.bfloat16, device="cuda") for _ in range(2))
        s.cache.read(0, new + 2, cu, s.table, kv_len, k=ko, v=vo)
        for got, x in ((ko, s.k[1]), (vo, s.v[1])):
            assert bool((got[:new] == 9.0).all()), f"{new} rows, kv_len {length}"
            assert torch.equal(got[new:].double(), stored(x[-2:], fmt))
        with pytest.raises(mp.MagicPigError, match="MP_ERR_DATA.*kv_len"):
            s.cache.check()
    s.compare(*s.attend())


@pytest.mark.gpu
def test_check_names_all_that_was_met_and_forgets_it():
    s = Setup([(1, 100), (2, 90)], 16, 8, 2, 128, "bf16", seed=19).fill()
    t, n = s.table.clone(), s.kv_len.clone()
    t[1, 0], n[0] = -1, 113
    for _ in range(2):
        s.cache.attention(0, s.q, s.cu, t, n)
        with pytest.raises(mp.MagicPigError, match="kv_len.*page id"):
            s.cache.check()
        s.cache.check()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        s.cache.read(0, 3, s.cu, s.table, n)
        with pytest.raises(mp.MagicPigError, match="kv_len"):
            s.cache.check()
    s.cache.check()
    s.compare(*s.attend())


@pytest.mark.gpu
def test_no_new_rows():
    s = Setup([(0, 100), (0, 3)], 16, 8, 2, 128, "bf16").fill()
    out, lse = s.attend()
    assert out.shape == (0, 8, 128) and lse.shape == (0, 8)
    k, v = s.cache.read(0, 0, s.cu, s.table, s.kv_len)
    assert k.shape == v.shape == (0, 2, 128)


# ---------------------------------------------------------------- refusals: nothing reaches the GPU
@pytest.mark.parametrize("change,code", [
    (dict(D=96), 5), (dict(H=7), 1), (dict(H=1), 1), (dict(layers=0), 1), (dict(pages=0), 1), (dict(pages=1 << 31), 1),
    (dict(size=0), 1), (dict(size=48), 1), (dict(size=8192), 1), (dict(size=-64), 1), (dict(fmt=2), 1), (dict(fmt=-1), 1),
    (dict(pages=(1 << 31) - 1, size=4096), 4)])
def test_refusals_of_alloc(change, code):
    h = C.c_void_p()
    assert L.lib().mp_paged_create(C.byref(h)) == 0
    a = {**dict(layers=1, H=8, Hkv=2, D=128, pages=4, size=64, fmt=0), **change}
    assert L.lib().mp_paged_alloc(h, *a.values()) == code
    assert b"mp_paged_alloc" in L.lib().mp_last_error()
    x = 1 << 20
    lib = L.lib()
    assert lib.mp_paged_append(h, 0, x, 256, 128, x, 256, 128, x, 1, 1, x, 1, x, None) == 2          # not allocated
    assert lib.mp_paged_read(h, 0, x, x, x, 1, 1, x, 1, x, None) == 2
    assert lib.mp_paged_attention(h, 0, x, 1024, 128, x, 1, 1, x, 1, x, 0.1, x, x, None, 0, None) == 2
    assert lib.mp_paged_workspace(h, 1, 1, 1, C.byref(C.c_int64())) == 2
    assert lib.mp_paged_check(h, None) == 2
    assert lib.mp_paged_destroy(h) == 0


def test_refusals_without_a_handle():
    lib, x = L.lib(), 1 << 20
    assert lib.mp_paged_create(None) == 1
    assert lib.mp_paged_alloc(None, 1, 8, 2, 128, 4, 64, 0) == 1
    assert lib.mp_paged_check(None, None) == 2
    assert lib.mp_paged_append(None, 0, x, 256, 128, x, 256, 128, x, 1, 1, x, 1, x, None) == 2
    assert lib.mp_paged_destroy(None) == 0
    with pytest.raises(ValueError, match="kv_format"):
        mp.PagedKVCache().alloc(1, 8, 2, 128, 4, 64, kv_format="int8")


@pytest.mark.gpu
@pytest.mark.parametrize("pairs,H,Hkv", [([(1, 9000), (5, 700)], 8, 2), ([(300, 4000), (1, 600)], 32, 8), ([(2100, 2300), (1, 600)], 32, 8)],
                         ids=["few rows", "many rows", "most rows"])
def test_outputs_over_the_queries(pairs, H, Hkv):
    s = Setup(pairs, 16, H, Hkv, 128, "bf16", seed=26).fill()
    want = s.attend()
    out, lse = s.cache.attention(0, s.q, s.cu, s.table, s.kv_len, out=s.q)
    assert out is s.q and torch.equal(out, want[0]) and torch.equal(lse, want[1])
    room = torch.zeros(s.q.numel() + 64, dtype=torch.bfloat16, device="cuda")
    a, b = (room[i:i + s.q.numel()].view_as(s.q) for i in (0, 64))
    with pytest.raises(mp.MagicPigError, match="overlap"):
        s.cache.attention(0, a, s.cu, s.table, s.kv_len, out=b)
    with pytest.raises(mp.MagicPigError, match="overlap"):
        s.cache.attention(0, s.q, s.cu, s.table, s.kv_len, out=a, lse=room.view(torch.float32)[:s.T * H].view(s.T, H))
    k = torch.zeros((s.T, Hkv, 128), dtype=torch.bfloat16, device="cuda")
    with pytest.raises(mp.MagicPigError, match="overlap"):
        s.cache.read(0, s.T, s.cu, s.table, s.kv_len, k=k, v=k)


@pytest.mark.gpu
def test_a_scale_that_is_infinite_in_base_2_is_refused():
    s = Setup([(2, 100)], 16, 8, 2, 128, "bf16").fill()
    with pytest.raises(mp.MagicPigError, match="scale"):
        s.attend(scale=3e38)
    s.compare(*s.attend(scale=1e-20), scale=1e-20)


@pytest.mark.gpu
def test_forward_gradients_are_refused():
    s = Setup([(2, 100)], 16, 8, 2, 128, "bf16").fill()
    with torch.autograd.forward_ad.dual_level():
        q, k = (torch.autograd.forward_ad.make_dual(x, torch.ones_like(x)) for x in (s.q, s.k[0][:2]))
        with pytest.raises(ValueError, match="q: .*tangent"):
            s.cache.attention(0, q, s.cu, s.table, s.kv_len)
        with pytest.raises(ValueError, match="v: .*tangent"):
            s.cache.append(0, s.k[0][:2], k, s.cu, s.table, s.kv_len)
    leaf = torch.empty((2, 2, 128), dtype=torch.bfloat16, device="cuda", requires_grad=True)
    with pytest.raises(ValueError, match="k: requires a gradient"):
        s.cache.read(0, 2, s.cu, s.table, s.kv_len, k=leaf)
    with pytest.raises(ValueError, match="out: requires a gradient"):
        s.attend(out=torch.empty_like(s.q).requires_grad_())


@pytest.mark.gpu
def test_refusals_of_calls():
    s = Setup([(2, 100)], 16, 8, 2, 128, "bf16").fill()
    c, k, cu, t, n = s.cache, s.k[0][:2], s.cu, s.table, s.kv_len
    with pytest.raises(mp.MagicPigError, match="layer_id"):
        c.append(1, k, k, cu, t, n)
    with pytest.raises(mp.MagicPigError, match="already allocated"):
        c.alloc(1, 8, 2, 128, 4, 64)
    with pytest.raises(mp.MagicPigError, match="aligned"):
        c.append(0, torch.zeros(600, dtype=torch.bfloat16, device="cuda")[1:513].view(2, 2, 128), k, cu, t, n)
    with pytest.raises(mp.MagicPigError, match="multiples of 8"):
        c.append(0, torch.zeros((2, 2, 130), dtype=torch.bfloat16, device="cuda")[:, :, :128], k, cu, t, n)
    with pytest.raises(ValueError, match="contiguous"):
        c.append(0, torch.zeros((2, 2, 256), dtype=torch.bfloat16, device="cuda")[:, :, ::2], k, cu, t, n)
    with pytest.raises(ValueError, match="cu_seqlens"):
        c.append(0, k, k, cu[:1], t, n)
    with pytest.raises(TypeError, match="page_table"):
        c.append(0, k, k, cu, t.long(), n)
    with pytest.raises(ValueError, match="kv_len: on cpu"):
        c.append(0, k, k, cu, t, n.cpu())
    with pytest.raises(ValueError, match="shape"):
        c.attention(0, s.q[:, :4], cu, t, n)
    with pytest.raises(mp.MagicPigError, match="scale"):
        s.attend(scale=-1.0)
    with pytest.raises(ValueError, match="out"):
        s.attend(out=torch.empty((2, 8, 64), dtype=torch.bfloat16, device="cuda"))
    long = Setup([(1, 9000)], 64, 8, 2, 128, "bf16").fill()
    need = C.c_int64()
    L.check(L.lib().mp_paged_workspace(long.cache._h, 1, 1, long.table.shape[1], C.byref(need)))
    assert need.value > 0
    for tokens in ((1 << 26) + 1, (1 << 63) - 1):
        assert L.lib().mp_paged_workspace(long.cache._h, 1, tokens, 1, C.byref(C.c_int64())) == 5      # as the call itself
        assert L.lib().mp_paged_append(long.cache._h, 0, 16, 256, 128, 16, 256, 128, 16, 1, tokens, 16, 1, 16, None) == 5
    o = torch.empty_like(long.q)
    for ptr, size in ((None, 0), (o.data_ptr(), need.value - 1), (o.data_ptr() + 8, need.value)):
        assert L.lib().mp_paged_attention(long.cache._h, 0, L.ptr(long.q), 1024, 128, L.ptr(long.cu), 1, 1, L.ptr(long.table),
                                          long.table.shape[1], L.ptr(long.kv_len), 0.1, L.ptr(o), None, ptr, size, None) == 1
