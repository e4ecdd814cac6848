"""Attention of grouped heads in 64 bits, with the error a kernel may make: every bf16 weight and every bf16 output is off by
at most 2^-8 of itself, f32 logits by their D products' roundings."""
import math

import torch

BF16 = torch.finfo(torch.bfloat16).eps / 2
F32 = torch.finfo(torch.float32).eps / 2


def attend(q, k, v, scale, lim):
    """q [n, H, D], k, v [c, Hkv, D]; query i sees keys 0 .. lim[i] (none below 0).  Returns out, lse (base 2) in f64 and the
    bounds of their errors.  Masked keys and values are not looked at, whatever they hold."""
    n, H, D = q.shape
    c, Hkv = k.shape[0], k.shape[1]
    out, tol = (torch.zeros((n, H, D), dtype=torch.float64, device=q.device) for _ in range(2))
    lse, ltol = (torch.full((n, H), x, dtype=torch.float64, device=q.device) for x in (float("-inf"), 0.0))
    see = torch.arange(c, device=q.device)[None, :] <= lim.to(q.device)[:, None]
    rows = see.any(1)
    if not bool(rows.any()):
        return out, tol, lse, ltol
    for h in range(H):
        kh, vh, qh = k[:, h * Hkv // H].double(), v[:, h * Hkv // H].double(), q[:, h].double()
        x = (qh @ torch.nan_to_num(kh, 0.0, 0.0, 0.0).t()) * scale
        odd = ~torch.isfinite(kh).all(1)
        if bool(odd.any()):                      # what a visible key with an infinity or NaN gives
            x[:, odd] = torch.stack([(qh * kh[j]).sum(1) * scale for j in odd.nonzero().flatten()], 1)
        x = torch.where(see, x, float("-inf"))
        z = torch.logsumexp(x, 1)
        p = torch.where(see, torch.exp(x - z[:, None]), 0.0)
        fine = torch.isfinite(vh)
        o = p @ torch.where(fine, vh, 0.0)
        mag = p @ torch.where(fine, vh.abs(), 0.0)
        for j in (~fine).any(1).nonzero().flatten():      # 0 of it where it is masked, else its infinity or NaN
            bad = torch.where(fine[j], 0.0, vh[j])
            o = o + torch.where(see[:, j, None], bad[None, :].expand_as(o), 0.0)
        dots = torch.where(see, (qh.abs() @ torch.nan_to_num(kh, 0.0, 0.0, 0.0).abs().t()) * scale, 0.0).amax(1)
        logit = dots * (D + 4) * F32                       # of a logit, absolute, natural units
        sums = (see.sum(1) + 64) * F32                     # of the f32 sums and of 2^x
        out[:, h], lse[:, h] = torch.where(rows[:, None], o, 0.0), torch.where(rows, z / math.log(2.0), float("-inf"))
        tol[:, h] = BF16 * (o.abs() + mag) * (1 + BF16) + (2 * logit + 2 * sums)[:, None] * mag + 1e-30
        ltol[:, h] = (logit + sums) / math.log(2.0) + z.abs().nan_to_num(0.0, 0.0, 0.0) * 4 * F32
    return out, tol, lse, ltol


def check(got, want, tol, what=""):
    """Equal where `want` is no finite number, within tol elsewhere."""
    got, want = got.double(), want.double()
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what + ": NaN in other places"
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf]), what + ": infinities differ"
    far = ((got - want).abs() - tol)[fine]
    assert far.numel() == 0 or bool((far <= 0).all()), f"{what}: off by {far.max().item():.3e} more than the bound"
