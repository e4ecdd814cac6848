"""Cases, plain forms and 64-bit references of the prompt and paged-cache operators.

Three operators, as a server that holds whole prompts and grows them chunk by chunk uses them:

    prompt   causal attention over whole prompts packed one behind the other (grouped heads)
    cache    new tokens written into a paged cache (bf16, or e4m3 with one power of two per row) and read back
    chunk    attention of each request's new tokens over its pages: one token of a decode step up to a prompt's chunk

`own` false: elementary torch operations in 32 bits.  `own` true: the calls of magicpig_amd a user makes.
"""
import math

import torch

own = False

DEV = "cuda"
CHUNK_ELEMS = 1 << 29          # scores of one block of the plain forms, elements


def listed():
    return [
        # one short question, an 8B model's heads: the smallest prompt call
        dict(name="prompt_short", op="prompt", lens="100", H=32, Hkv=8, D=128, fused=0),
        # a batch of prompts of very different lengths, q | k | v slices of one projection
        dict(name="prompt_ragged", op="prompt", lens="1,17,64,129,3,700,2047,255,1024,4001,33,512,1,1500", H=32, Hkv=8, D=128, fused=1),
        # one rank's heads of a 70B model over 8 ranks, a long prompt
        dict(name="prompt_rank", op="prompt", lens="16384", H=8, Hkv=1, D=128, fused=0),
        # 64-wide heads, two documents
        dict(name="prompt_d64", op="prompt", lens="5000,3100", H=32, Hkv=8, D=64, fused=0),
        # a whole 32K prompt of the 8B model: the largest
        dict(name="prompt_long", op="prompt", lens="32768", H=32, Hkv=8, D=128, fused=0),
        # the cache's part of a decode step: one token of each of 8 requests
        dict(name="cache_step", op="cache", new="1*8", kv="32769*8", page=64, fmt="e4m3", Hkv=8, D=128),
        # a chunk of 2048 tokens behind 4096, one request, unquantised
        dict(name="cache_chunk", op="cache", new="2048", kv="6144", page=16, fmt="bf16", Hkv=8, D=128),
        # a whole 98 000-token prompt quantised as it is written
        dict(name="cache_prompt", op="cache", new="98000", kv="98000", page=64, fmt="e4m3", Hkv=8, D=128),
        # a decode step of one request behind 98 000 tokens
        dict(name="step_long", op="chunk", new="1", kv="98001", page=64, fmt="bf16", H=32, Hkv=8, D=128),
        # a decode step of a batch of 64 at uneven lengths over a quantised cache, one rank of 8 of a 70B model
        dict(name="step_batch", op="chunk", new="1*64", kv="1-8000*64", page=32, fmt="e4m3", H=8, Hkv=1, D=128),
        # drafted tokens of 8 requests behind 32K each, quantised
        dict(name="draft_batch", op="chunk", new="5*8", kv="32773*8", page=64, fmt="e4m3", H=32, Hkv=8, D=128),
        # one chunk of a long prompt that is prefilled piece by piece
        dict(name="chunk_long", op="chunk", new="2048", kv="67584", page=64, fmt="bf16", H=32, Hkv=8, D=128),
    ]


def log_uniform(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    op = rng.choice(["prompt", "cache", "chunk"])
    D = rng.choice([64, 128, 128])
    H, Hkv = rng.choice([(32, 8), (32, 8), (8, 1), (64, 8), (8, 8), (6, 2), (14, 2)])
    if op == "prompt":
        n = log_uniform(rng, 1, 32)
        budget = 32768 if n == 1 and H <= 32 else 16384
        lens = [log_uniform(rng, 1, max(1, budget // n)) for _ in range(n)]
        return dict(op=op, lens=",".join(map(str, lens)), H=H, Hkv=Hkv, D=D, fused=rng.randint(0, 1))
    page = rng.choice([1, 8, 16, 32, 64, 128, 256])
    fmt = rng.choice(["bf16", "e4m3"])
    n = log_uniform(rng, 1, 64)
    kv = [log_uniform(rng, 1, max(1, 98000 // n)) for _ in range(n)]
    if op == "cache":
        new = [log_uniform(rng, 1, c) for c in kv]
        return dict(op=op, new=",".join(map(str, new)), kv=",".join(map(str, kv)), page=page, fmt=fmt, Hkv=Hkv, D=D)
    top = rng.choice([1, 1, 8, max(1, 1024 // n)])
    new = [min(c, log_uniform(rng, 1, top)) for c in kv]
    return dict(op=op, new=",".join(map(str, new)), kv=",".join(map(str, kv)), page=page, fmt=fmt, H=H, Hkv=Hkv, D=D)


def lengths(text):
    """"3,17", "1*8" (8 times 1) or "1-8000*64" (64 lengths spread evenly from 1 to 8000)."""
    out = []
    for part in text.split(","):
        size, _, times = part.partition("*")
        lo, _, hi = size.partition("-")
        n = int(times or 1)
        out += [int(lo) if not hi else int(lo) + (int(hi) - int(lo)) * i // max(1, n - 1) for i in range(n)]
    return out


def offsets(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return out


def inputs(case, seed):
    """Everything both forms start from, on the GPU."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    Hkv, D = case["Hkv"], case["D"]

    def rows(n, heads, spread=1.0, mean=None):
        x = torch.randn((n, heads, D), generator=g, device=DEV) * spread
        return (x if mean is None else x + mean).to(torch.bfloat16)

    kmean = torch.randn((1, Hkv, D), generator=g, device=DEV) * 2.0    # keys have a common part, channel by channel
    if case["op"] == "prompt":
        lens = lengths(case["lens"])
        T, H = sum(lens), case["H"]
        q, k, v = rows(T, H, 1.5), rows(T, Hkv, 1.0, kmean), rows(T, Hkv)
        if case["fused"]:
            qkv = torch.cat([q, k, v], dim=1)
            q, k, v = qkv[:, :H], qkv[:, H:H + Hkv], qkv[:, H + Hkv:]
        return dict(case=case, lens=lens, q=q, k=k, v=v,
                    cu=torch.tensor(offsets(lens), dtype=torch.int32, device=DEV))
    new, kv, page = lengths(case["new"]), lengths(case["kv"]), case["page"]
    per = [-(-c // page) for c in kv]
    P, pages = max(per), sum(per)
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)     # pages in no order
    table = torch.zeros((len(kv), P), dtype=torch.int32, device=DEV)
    for b, first in enumerate(offsets(per)[:-1]):
        table[b, :per[b]] = order[first:first + per[b]]
    s = dict(case=case, new=new, kv=kv, table=table, pages=pages, cu=torch.tensor(offsets(new), dtype=torch.int32, device=DEV),
             kv_len=torch.tensor(kv, dtype=torch.int32, device=DEV))
    n = sum(new) if case["op"] == "cache" else sum(kv)
    s["k"], s["v"] = rows(n, Hkv, 1.0, kmean), rows(n, Hkv)
    if case["op"] == "chunk":
        s["q"] = rows(sum(new), case["H"], 1.5)
        s["cu_all"] = torch.tensor(offsets(kv), dtype=torch.int32, device=DEV)
    return s


def slots(table, page, first, last, b):
    """Rows of the flat cache [pages * page] that hold positions first..last-1 of request b."""
    pos = torch.arange(first, last, device=DEV)
    return table[b].long()[pos // page] * page + pos % page


def all_slots(s, new, kv):
    return torch.cat([slots(s["table"], s["case"]["page"], c - n, c, b) for b, (n, c) in enumerate(zip(new, kv))])


def prepare(case, seed):
    s = inputs(case, seed)
    if case["op"] == "prompt":
        return s
    Hkv, D, page = case["Hkv"], case["D"], case["page"]
    if own:
        import magicpig_amd

        cache = magicpig_amd.PagedKVCache()
        cache.alloc(1, case.get("H", Hkv), Hkv, D, s["pages"], page, kv_format=case["fmt"])
        s["cache"] = cache
        if case["op"] == "chunk":
            cache.append(0, s.pop("k"), s.pop("v"), s["cu_all"], s["table"], s["kv_len"])
        return s
    rows = s["pages"] * page
    if case["fmt"] == "bf16":
        s["pool"] = torch.zeros((rows, Hkv, 2, D), dtype=torch.bfloat16, device=DEV)
    else:
        s["pool"] = torch.zeros((rows, Hkv, 2, D), dtype=torch.float8_e4m3fn, device=DEV)
        s["power"] = torch.zeros((rows, Hkv, 2, 1), dtype=torch.int32, device=DEV)
    if case["op"] == "chunk":
        plain_write(s, s.pop("k"), s.pop("v"), all_slots(s, s["kv"], s["kv"]))
    return s


def power_of_two(e):
    """2^e in 32 bits, from its bits: a power function may be off in the last one."""
    return ((e.int() + 127) << 23).view(torch.float32)


# ---------------------------------------------------------------- plain forms
def plain_write(s, k, v, where):
    x = torch.stack([k, v], dim=2)
    if s["case"]["fmt"] == "bf16":
        s["pool"][where] = x
        return
    x = x.float()
    # the least e with max|x| <= 448 * 2^e: every later product with 2^e is exact
    m, e = torch.frexp(x.abs().amax(-1, keepdim=True))
    e = (e - 9 + (m > 0.875).int()).clamp(min=-126)
    s["pool"].view(torch.uint8)[where] = (x * power_of_two(-e)).to(torch.float8_e4m3fn).view(torch.uint8)
    s["power"][where] = e


def plain_read(s, where):
    """f32 [n, Hkv, 2, D]: what the rows stand for."""
    if s["case"]["fmt"] == "bf16":
        return s["pool"][where].float()
    x = s["pool"].view(torch.uint8)[where].view(torch.float8_e4m3fn).float()
    return x * power_of_two(s["power"][where])


def plain_attention(q, k, v):
    """q [n, H, D], k, v [c, Hkv, D], all f32: query i sees keys 0 .. c - n + i.  Returns out, base-2 log-sum-exp."""
    n, H, D = q.shape
    c, Hkv = k.shape[0], k.shape[1]
    G = H // Hkv
    out = torch.empty((n, H, D), dtype=q.dtype, device=q.device)
    lse = torch.empty((n, H), dtype=q.dtype, device=q.device)
    step = max(1, CHUNK_ELEMS // (c * G))
    for h in range(Hkv):
        kt, vh = k[:, h].t().contiguous(), v[:, h].contiguous()
        for i in range(0, n, step):
            j = min(n, i + step)
            seen = c - n + j
            x = q[i:j, h * G:(h + 1) * G].reshape(-1, D) @ kt[:, :seen]
            x = (x * (D ** -0.5)).view(j - i, G, seen)
            last = torch.arange(c - n + i, c - n + j, device=q.device).view(-1, 1, 1)
            x.masked_fill_(torch.arange(seen, device=q.device) > last, float("-inf"))
            top = x.amax(-1, keepdim=True)
            x.sub_(top).exp_()
            total = x.sum(-1, keepdim=True)
            y = (x.view(-1, seen) @ vh[:seen]).view(j - i, G, D) / total
            out[i:j, h * G:(h + 1) * G] = y
            lse[i:j, h * G:(h + 1) * G] = ((top + total.log()) * math.log2(math.e)).squeeze(-1)
    return out, lse


def plain(s):
    case = s["case"]
    if case["op"] == "cache":
        where = all_slots(s, s["new"], s["kv"])
        plain_write(s, s["k"], s["v"], where)
        x = plain_read(s, where).to(torch.bfloat16)
        return x[:, :, 0], x[:, :, 1]
    outs, lses = [], []
    if case["op"] == "prompt":
        ends = offsets(s["lens"])
        for a, b in zip(ends, ends[1:]):
            o, l = plain_attention(s["q"][a:b].float(), s["k"][a:b].float(), s["v"][a:b].float())
            outs.append(o.to(torch.bfloat16))
            lses.append(l)
    else:
        ends = offsets(s["new"])
        for b, c in enumerate(s["kv"]):
            x = plain_read(s, slots(s["table"], case["page"], 0, c, b))
            o, l = plain_attention(s["q"][ends[b]:ends[b + 1]].float(), x[:, :, 0], x[:, :, 1])
            outs.append(o.to(torch.bfloat16))
            lses.append(l)
    return torch.cat(outs), torch.cat(lses)


def run(s):
    if not own:
        return plain(s)
    import magicpig_amd

    op = s["case"]["op"]
    if op == "prompt":
        return magicpig_amd.prompt_attention(s["q"], s["k"], s["v"], s["cu"])
    if op == "cache":
        s["cache"].append(0, s["k"], s["v"], s["cu"], s["table"], s["kv_len"])
        return s["cache"].read(0, s["k"].shape[0], s["cu"], s["table"], s["kv_len"])
    return s["cache"].attention(0, s["q"], s["cu"], s["table"], s["kv_len"])


# ---------------------------------------------------------------- 64 bits
def quantised(x):
    """What e4m3 rows of x stand for, in 64 bits: 3 bits behind the point, least exponent -6, ties to even."""
    x = x.double()

    def floor_power(a):                                  # 2^floor(log2 a) of normal a > 0: its exponent bits alone
        return (a.view(torch.int64) & (0x7FF << 52)).view(torch.float64)

    top = x.abs().amax(-1, keepdim=True).clamp(min=2.0 ** -200)
    scale = floor_power(top) * 2.0 ** -8                 # 448 = 1.75 * 2^8
    scale = torch.where(top > 448.0 * scale, scale * 2.0, scale).clamp(min=2.0 ** -126)
    y = x / scale
    unit = floor_power(y.abs().clamp(min=2.0 ** -6)) * 0.125
    return torch.round(y / unit) * unit * scale


def exact_attention(q, k, v):
    """The same sums as a definition: one query block and one query head at a time."""
    n, H, D = q.shape
    c, Hkv = k.shape[0], k.shape[1]
    out = torch.empty((n, H, D), dtype=torch.float64, device=DEV)
    lse = torch.empty((n, H), dtype=torch.float64, device=DEV)
    block = max(1, (1 << 27) // c)
    for h in range(H):
        kh, vh = k[:, h * Hkv // H].double(), v[:, h * Hkv // H].double()
        for i in range(0, n, block):
            rows = torch.arange(i, min(n, i + block), device=DEV)
            seen = int(c - n + rows[-1] + 1) if n > 1 else c
            w = torch.matmul(q[rows, h].double(), kh[:seen].t()) / math.sqrt(D)
            w = torch.where(torch.arange(seen, device=DEV)[None, :] <= (c - n + rows)[:, None], w, float("-inf"))
            z = torch.logsumexp(w, dim=1)
            out[rows, h] = torch.matmul(torch.exp(w - z[:, None]), vh[:seen])
            lse[rows, h] = z / math.log(2.0)
    return out, lse


def exact(case, seed):
    s = inputs(case, seed)
    if case["op"] == "cache":
        if case["fmt"] == "bf16":
            return s["k"].double(), s["v"].double()
        return quantised(s["k"]), quantised(s["v"])
    if work(case)["flops"] > 1.5e13:       # more than about 20 s
        return None
    parts = []
    ends = offsets(s["lens"] if case["op"] == "prompt" else s["new"])
    if case["op"] == "prompt":
        for a, b in zip(ends, ends[1:]):
            parts.append(exact_attention(s["q"][a:b], s["k"][a:b], s["v"][a:b]))
    else:
        stored = (lambda x: x) if case["fmt"] == "bf16" else quantised
        begin = offsets(s["kv"])
        for b in range(len(s["kv"])):
            k, v = s["k"][begin[b]:begin[b + 1]], s["v"][begin[b]:begin[b + 1]]
            parts.append(exact_attention(s["q"][ends[b]:ends[b + 1]], stored(k), stored(v)))
    return torch.cat([p[0] for p in parts]), torch.cat([p[1] for p in parts])


def work(case):
    Hkv, D = case["Hkv"], case["D"]
    row = 2 * D * 2 if case.get("fmt", "bf16") == "bf16" else 2 * D + 2       # one head's K and V of a token in the cache
    if case["op"] == "cache":
        new = sum(lengths(case["new"]))
        # new rows in, their cache rows out and in again, read-back rows out
        return dict(bytes=new * Hkv * (2 * 4 * D + 2 * row), flops=new * Hkv * 4 * D)
    H = case["H"]
    if case["op"] == "prompt":
        lens = lengths(case["lens"])
        pairs, new, kv_bytes = sum(n * (n + 1) // 2 for n in lens), sum(lens), sum(lens) * Hkv * 4 * D
    else:
        n, kv = lengths(case["new"]), lengths(case["kv"])
        pairs, new = sum(a * (c - a) + a * (a + 1) // 2 for a, c in zip(n, kv)), sum(n)
        kv_bytes = sum(kv) * Hkv * row
    return dict(bytes=kv_bytes + new * H * (4 * D + 4), flops=4 * pairs * H * D)
