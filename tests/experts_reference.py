"""Plain 64-bit forms of the mixture-of-experts operators, with error bounds.

Bounds.  A rounding to bf16 is off by at most 2^-8 of the value (half of finfo.eps), one to e4m3 by
at most 2^-4 of it, or 2^-10 of the block's scale below the smallest normal.  A sum of n products in
fp32 is off by at most n * 2^-23 * sum|products| (every product of two bf16 values is exact; one
rounding or truncation per addition).  The activation's ex2 and rcp are off by less than 2^-21
together, which 2^-20 covers with the three multiplications that follow.
"""
import torch

BF16_HALF = 2.0 ** -8
E4M3_HALF = 2.0 ** -4
ACC = 2.0 ** -23
ACT = 2.0 ** -20
TINY = 2.0 ** -100       # results below may be flushed (approximate reciprocal)


def order(ids, E):
    """(offsets, slots, rows) by a plain loop."""
    T, k = ids.shape
    flat = ids.reshape(-1).tolist()
    by = [[] for _ in range(E)]
    for s, e in enumerate(flat):
        if 0 <= e < E:
            by[e].append(s)
    offsets, slots = [0], []
    for b in by:
        slots += b
        offsets.append(len(slots))
    rows = [-1] * len(flat)
    for r, s in enumerate(slots):
        rows[s] = r
    slots += [-1] * (len(flat) - len(slots))
    return (torch.tensor(offsets, dtype=torch.int32), torch.tensor(slots, dtype=torch.int32),
            torch.tensor(rows, dtype=torch.int32).view(T, k))


def product(a, b):
    """a @ b in 64 bits, and the bound on the fp32 sum."""
    a, b = a.double(), b.double()
    return a @ b, a.shape[1] * ACC * (a.abs() @ b.abs())


def silu(g):
    return g * torch.sigmoid(g)


def silu_grad(g):
    s = torch.sigmoid(g)
    return s * (1 + g * (1 - s))


def swiglu(x, w):
    """(h, bound of h before its rounding, up, bound, gate, bound)"""
    n = w.shape[1] // 2
    up, du = product(x, w[:, :n])
    gate, dg = product(x, w[:, n:])
    h = up * silu(gate)
    # |silu'| < 1.1; both factors may be off at once
    bound = silu(gate).abs() * du + 1.1 * (up.abs() + du) * dg + ACT * h.abs()
    return h, bound, up, du, gate, dg


def rounded(value, bound):
    """The bound after the result was rounded to bf16."""
    return bound + BF16_HALF * (value.abs() + bound) + TINY


def assert_within(got, want, bound, what=""):
    got = got.double().to(want.device)
    bad = ~((got - want).abs() <= bound)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} outside, first at "
                           f"{bad.nonzero()[0].tolist()}: got {got[bad][0].item()!r} want "
                           f"{want[bad][0].item()!r} bound {bound[bad][0].item():.3g}")


def block_codes(v):
    """e4m3 codes [rows, blocks * 32] and scale codes [rows, blocks] of fp32 values that are known
    exactly (columns padded with zeros)."""
    rows, n = v.shape
    b = torch.nn.functional.pad(v.double(), (0, -n % 32)).view(rows, -1, 32)
    top = b.abs().amax(-1)
    e = torch.full(top.shape, -127, dtype=torch.int64)
    for i in range(-127, 121):          # the smallest exponent that holds the block's maximum
        e = torch.where(448.0 * 2.0 ** (i - 1) < top, torch.full_like(e, i), e)
    q = (b * torch.exp2(-e.double())[..., None]).float().to(torch.float8_e4m3fn)
    return q.view(torch.uint8).view(rows, -1), (e + 127).to(torch.uint8)


def saved_values(pre):
    """(up, gate) in 64 bits that a SavedPreact stands for."""
    if pre.bits == 16:
        v = pre.data[..., :pre.hidden].double()
    else:
        nb = (pre.hidden + 31) // 32
        scale = torch.exp2(pre.scales[..., :nb].double() - 127)
        scale = torch.where(pre.scales[..., :nb] == 255, torch.nan, scale)
        v = pre.data.view(torch.float8_e4m3fn).to(torch.float32).double()
        v = (v.unflatten(-1, (-1, 32)) * scale[..., None]).flatten(-2)[..., :pre.hidden]
    return v[:, 0], v[:, 1]
