"""The operators of the 8-bit path in 64 bits, for the tests: the definitions, and how far a 32-bit evaluation may be from them.

Bounds count roundings: u = 2^-24 is half a step of float32, a sum of n terms in any order is off by at most n u times the
sum of the magnitudes, a rounding to type t by at most finfo(t).eps / 2 of the value.  Matrix-core sums are given 2 u per
addition (they may truncate)."""
import torch

U = 2.0 ** -24
GROUP, E4M3_MAX, FLOOR = 128, 448.0, 1e-10


def groups(n):
    return -(-n // GROUP)


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def smallest(dtype):
    """Half a step below the smallest normal number (where a rounding is absolute, not relative)."""
    return torch.finfo(dtype).smallest_normal * half_step(dtype)


def spread_scale(scale, cols, rows=None):
    s = scale.double().repeat_interleave(GROUP, -1)[..., :cols]
    if rows is not None:
        s = s.repeat_interleave(GROUP, -2)[..., :rows, :]
    return s


def quant_scale(v):
    """[T, C] in 64 bits -> the scale of each group."""
    t, c = v.shape
    p = torch.zeros(t, groups(c) * GROUP, dtype=torch.float64, device=v.device)
    p[:, :c] = v
    return p.view(t, -1, GROUP).abs().amax(2).clamp(min=FLOOR) / E4M3_MAX


def check_quantized(q, scale, v, rel):
    """q, scale against the exact values v, which a 32-bit evaluation has to `rel` of themselves."""
    want = quant_scale(v)
    assert bool(((scale.double() - want).abs() <= want * (rel + 2 * U)).all()), "scales"
    s = spread_scale(scale, v.shape[1])
    off = (q.double() * s - v).abs()
    # half a step of e4m3: 2^-4 of the value, or 2^-10 scales below its smallest normal number; the quotient's own roundings
    allowed = v.abs() * (2.0 ** -4 + rel + 8 * U) + s * 2.0 ** -10 * (1 + 8 * U)
    assert bool((off <= allowed).all()), f"8-bit values: {(off - allowed).max().item()}"


def norm64(x, residual, weight, eps):
    r = x.double() if residual is None else x.double() + residual.double()
    return r, r / (r.square().mean(1, keepdim=True) + eps).sqrt() * weight.double()


# the norm in 32 bits: the sum x + residual (1 rounding), squares and their sum (at most 64 + 8 + 16 roundings deep, halved by the
# root), the mean, eps, root and reciprocal, two products
NORM_REL = (1 + 2 * 1 + (88 + 2) / 2 + 4 + 2) * U


def swiglu64(gate_up):
    i = gate_up.shape[1] // 2
    g, u = gate_up[:, :i].double(), gate_up[:, i:].double()
    return g * torch.sigmoid(g) * u


# expf to 2 ulp (4 u), 1 + e, the quotient (to 1 ulp), the product
SWIGLU_REL = (4 + 1 + 2 + 1) * U


def widen(w, scale, block_rows):
    """e4m3 weights (or rows, block_rows False) and their scales in 64 bits."""
    if scale is None:
        return w.double()
    return w.double() * spread_scale(scale, w.shape[-1], w.shape[-2] if block_rows else None)


def dropped(wa, wb):
    """What the 8-bit matrix instruction may drop: of 8 neighbouring products everything more than 13 bits below the largest, so
    of each less than 2^-13 of the largest."""
    total = torch.zeros(wa.shape[0], wb.shape[0], dtype=torch.float64, device=wa.device)
    for at in range(0, wa.shape[1], 8):
        most = torch.zeros_like(total)
        for k in range(at, min(at + 8, wa.shape[1])):
            torch.maximum(most, wa[:, k].abs()[:, None] * wb[:, k].abs()[None, :], out=most)
        total += most
    return total * 8 * 2.0 ** -13


def check_matmul(c, a, a_scale, b, b_scale):
    k = a.shape[1]
    wa, wb = widen(a, a_scale, False), widen(b, b_scale, True)
    want, size = wa @ wb.t().contiguous(), wa.abs() @ wb.abs().t().contiguous()
    # 128 terms of a group and the groups' sums, 2 u each; the scales' product and its product with the sum
    allowed = want.abs() * half_step(c.dtype) + size * (2 * (min(k, GROUP) + groups(k)) + 4) * U + smallest(c.dtype)
    if c.dtype is not torch.float32:
        allowed += dropped(wa, wb) * (1 + half_step(c.dtype))
    off = (c.double() - want).abs()
    # beyond the type's range (its largest number and half a step) a rounding gives infinity
    over = torch.isinf(c) & (want.abs() + allowed >= torch.finfo(c.dtype).max * (1 + half_step(c.dtype))) & (torch.sign(c.double()) == torch.sign(want))
    off[over] = 0
    want = torch.where(over, torch.zeros_like(want), want)
    assert bool((off <= allowed).all()), f"off by up to {(off / allowed.clamp_min(1e-300)).max().item()} of what is allowed"
    if c.dtype is not torch.float32 and want.numel() >= 256:
        # ... and taken together, where what is dropped is random, no more than 2^-14 (on normal data 1.4e-5 was measured) beside the rounding
        assert (off.norm() / want.norm()).item() <= half_step(c.dtype) + 2.0 ** -14
    return want


def choice(logits, topk):
    """Indices of the topk largest of each row, equal ones by rising index; a NaN counts as larger than any number."""
    key = logits.double().clone()
    key[torch.isnan(key)] = float("inf")
    key = torch.where(torch.isnan(logits), torch.full_like(key, 1e300), torch.where(torch.isinf(key) & (key > 0), torch.full_like(key, 1e299), key))
    return torch.sort(key, dim=1, descending=True, stable=True).indices[:, :topk]


def probabilities(logits, ids, renormalize):
    l = logits.double()
    top = l.gather(1, ids)
    p = torch.softmax(top, 1) if renormalize else torch.softmax(l, 1).gather(1, ids)
    dead = torch.isinf(top) & (top < 0)
    return torch.where(dead, torch.zeros_like(p), p)


def moe64(x, logits, topk, w13, w2, s13, s2, renormalize):
    """-> (out, how far a 32-bit evaluation may be from it before the last rounding, ids, probs)."""
    t, h = x.shape
    i = w2.shape[2]
    ids = choice(logits, topk)
    probs = probabilities(logits, ids, renormalize)
    out = torch.zeros(t, h, dtype=torch.float64, device=x.device)
    err = torch.zeros_like(out)
    xd = x.double()
    for e in sorted(set(ids.flatten().tolist())):
        a, b = widen(w13[e], None if s13 is None else s13[e], True), widen(w2[e], None if s2 is None else s2[e], True)
        rows = (ids == e).nonzero()
        for tok, j in rows.tolist():
            p = probs[tok, j]
            if p == 0:
                continue
            v, size = a @ xd[tok], a.abs() @ xd[tok].abs()
            g, u = v[:i], v[i:]
            sig = torch.sigmoid(g)
            hh = g * sig * u
            dv = size * (2 * (h + groups(h)) + 2 + 8) * U             # the products' sums, block scales, 8 waves
            # silu' <= 1.1; the activation's own roundings; two bf16 parts: 2^-9 of 2^-9
            dh = 1.1 * dv[:i] * u.abs() + (g * sig).abs() * dv[i:] + 1.1 * dv[:i] * dv[i:] + hh.abs() * (SWIGLU_REL + 2.0 ** -18)
            out[tok] += p * (b @ hh)
            # the second product's sums (twice the terms: two parts), then 16 partial sums and the places; p to a few roundings
            err[tok] += p * (b.abs() @ (dh + hh.abs() * (2 * (2 * i + groups(i) + 16 + topk) + 8 + 4 * 16) * U))
    return out, err, ids, probs
