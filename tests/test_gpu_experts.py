"""Mixture-of-experts operators and saved pre-activations against plain forms in 64 bits.
Tolerances are derived in ``experts_reference``."""
import pytest
import torch

import experts_reference as ref
import swiglu_fused_b200 as sg
from swiglu_fused_b200 import _lib

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16 = torch.bfloat16


@pytest.fixture(autouse=True)
def _device_status_clean():
    yield
    torch.cuda.synchronize()
    _lib.device_status()


def randn(*shape, seed=0, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * std).to(BF16).to(DEV)


def offsets_of(counts):
    return torch.tensor([0] + list(torch.tensor(counts).cumsum(0)), dtype=torch.int32, device=DEV)


def make_ids(T, k, E, seed, drop=0.1, dtype=torch.int64):
    g = torch.Generator().manual_seed(seed)
    ids = torch.randint(0, E, (T, k), generator=g)
    ids[torch.rand(T, k, generator=g) < drop] = -1
    return ids.to(dtype).to(DEV)


# ---------------------------------------------------------------- order


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("T,k,E,drop", [
    (1, 1, 1, 0.0), (1, 2, 8, 0.0), (1, 1, 4, 1.0), (7, 3, 5, 0.3), (33, 1, 1024, 0.0),
    (96, 8, 128, 0.0), (1000, 4, 3, 0.1), (2048, 2, 8, 0.0), (2049, 2, 8, 0.0), (4097, 3, 257, 0.2),
    (20000, 2, 1000, 0.05), (5000, 64, 64, 0.0), (100000, 6, 7, 0.3), (150000, 2, 1024, 0.0)])
def test_order(T, k, E, drop, dtype):
    ids = make_ids(T, k, E, T + k, drop, dtype)
    got = sg.expert_order(ids, E)
    for g, w, name in zip(got, ref.order(ids.cpu(), E), got._fields):
        assert torch.equal(g.cpu(), w), name


def test_order_ids_of_any_value_and_pitch():
    E = 6
    big = torch.tensor([[0, 5, 6], [-1, -2 ** 40, 2 ** 40], [5, 5, 5], [2 ** 32, 2 ** 32 + 1, 3]],
                       device=DEV)     # 2^32 is not expert 0
    wide = torch.full((4, 7), 1, dtype=torch.int64, device=DEV)
    wide[:, 2:5] = big
    want = ref.order(big.cpu(), E)
    for ids in (big, wide[:, 2:5]):
        for g, w in zip(sg.expert_order(ids, E), want):
            assert torch.equal(g.cpu(), w)
    # every slot of one expert; none of any
    one = torch.full((3000, 2), 4, device=DEV)
    for g, w in zip(sg.expert_order(one, E), ref.order(one.cpu(), E)):
        assert torch.equal(g.cpu(), w)
    none = torch.full((3000, 2), -1, device=DEV)
    for g, w in zip(sg.expert_order(none, E), ref.order(none.cpu(), E)):
        assert torch.equal(g.cpu(), w)


def test_no_tokens():
    ids = torch.empty((0, 2), dtype=torch.int64, device=DEV)
    order = sg.expert_order(ids, 4)
    assert order.offsets.tolist() == [0] * 5 and order.rows.shape == (0, 2)
    x = torch.empty((0, 16), dtype=BF16, device=DEV)
    assert sg.expert_dispatch(x, order).shape == (0, 16)
    assert sg.expert_combine(x, order).shape == (0, 16)
    w = randn(4, 16, 32)
    wd = randn(4, 16, 16)
    assert sg.grouped_fused_swiglu(x, w, order.offsets).shape == (0, 16)
    assert not sg.grouped_weight_grad(x, x, order.offsets).any()
    y = sg.experts_swiglu(x, ids, torch.empty((0, 2), device=DEV), w, wd)
    assert y.shape == (0, 16)
    for ck in ("bf16", "e4m3"):
        wg = w.clone().requires_grad_(True)
        sg.fused_swiglu_experts(x, ids, torch.empty((0, 2), device=DEV), wg, wd,
                                checkpoint=ck).sum().backward()
        assert not wg.grad.any()


# ---------------------------------------------------------------- rows out and back


@pytest.mark.parametrize("T,k,E,D,drop", [(1, 1, 1, 8, 0.0), (5, 3, 4, 8, 0.5), (333, 3, 10, 1416, 0.1),
                                          (64, 8, 16, 264, 0.0), (129, 2, 8, 4096, 0.2),
                                          (40, 11, 16, 72, 0.3), (3000, 2, 4, 136, 1.0)])
@pytest.mark.parametrize("wdtype", [torch.float32, BF16])
def test_dispatch_combine_and_gradients(T, k, E, D, drop, wdtype):
    ids = make_ids(T, k, E, T + D, drop)
    order = sg.expert_order(ids, E)
    R = T * k
    kept = int(order.offsets[-1])
    rows = order.rows.cpu()
    slots = order.slots.cpu()[:kept].long()
    x, ys, dy = randn(T, D, seed=1), randn(R, D, seed=2), randn(T, D, seed=3)
    gen = torch.Generator().manual_seed(4)
    w = torch.randn(T, k, generator=gen).to(wdtype).to(DEV)
    # dispatch: exact, strided, guarded
    wide = torch.full((R + 2, D + 16), 7.0, dtype=BF16, device=DEV)
    got = sg.expert_dispatch(x, order, out=wide[1:R + 1, 8:D + 8])
    assert torch.equal(got[:kept].cpu(), x.cpu()[slots // k])
    wide[1:kept + 1, 8:D + 8] = 7.0
    assert (wide == 7.0).all(), "wrote outside its rows"
    # combine
    on = (rows >= 0)
    picked = ys.cpu().double()[rows.clamp(min=0).long()] * on[..., None]
    for weights in (w, None):
        ww = (w.cpu().double() if weights is not None else torch.ones(T, k).double())[..., None]
        want = (picked * ww).sum(1)
        bound = ref.rounded(want, 2 * k * ref.ACC * (picked * ww).abs().sum(1))
        ref.assert_within(sg.expert_combine(ys, order, weights).cpu(), want, bound, "combine")
    # gradients
    buf = torch.full((R, D), 7.0, dtype=BF16, device=DEV)
    gys, gw = sg.expert_combine_grad(dy, ys, order, w, out=buf)
    want = dy.cpu().double()[slots // k] * w.cpu().double().reshape(-1)[slots][:, None]
    ref.assert_within(gys[:kept].cpu(), want, ref.rounded(want, ref.ACC * want.abs()), "grad_rows")
    assert (gys[kept:] == 7.0).all()
    prod = picked * dy.cpu().double()[:, None]
    want = prod.sum(-1)
    bound = D * ref.ACC * prod.abs().sum(-1)
    if wdtype == BF16:
        bound = ref.rounded(want, bound)
    ref.assert_within(gw.cpu(), want, bound + ref.TINY, "grad_weights")
    assert not gw.cpu()[~on].any() and gw.dtype == wdtype
    only, nothing = sg.expert_combine_grad(dy, None, order, w, out=torch.full_like(buf, 7.0))
    assert nothing is None and torch.equal(only, buf)
    # fp32 rows hold the same values; rows without the weights
    y32 = ys.float()
    assert torch.equal(sg.expert_combine(y32, order, w), sg.expert_combine(ys, order, w))
    plain, gw32 = sg.expert_combine_grad(dy, y32, order, w, weighted=False,
                                         out=torch.full_like(buf, 7.0))
    assert torch.equal(gw32, gw) and (plain[kept:] == 7.0).all()
    assert torch.equal(plain[:kept].cpu(), dy.cpu()[slots // k])
    inplace = ys.clone()
    sg.expert_combine_grad(dy, inplace, order, w, out=inplace)
    assert torch.equal(inplace[:kept], buf[:kept])


def test_combine_skips_dropped_slots_even_with_nan():
    ids = torch.tensor([[0, -1], [1, 0], [-1, -1]], device=DEV)
    order = sg.expert_order(ids, 2)
    ys = randn(6, 16)
    ys[3:] = float("nan")                       # rows that do not exist
    w = torch.tensor([[0.5, float("nan")], [1.0, 2.0], [float("inf"), float("nan")]], device=DEV)
    y = sg.expert_combine(ys, order, w)
    assert torch.isfinite(y).all() and not y[2].any()
    dy = randn(3, 16, seed=5)
    gys, gw = sg.expert_combine_grad(dy, ys, order, w, out=torch.zeros_like(ys))
    assert torch.isfinite(gys).all() and torch.isfinite(gw).all()


# ---------------------------------------------------------------- products

# groups: lone rows, empty groups, borders inside and on tiles, one group, large ones (CTA pairs)
GROUPS = [[1], [1, 0, 1], [0, 0, 5], [16, 17, 0, 15], [128, 128], [127, 1, 129, 0, 300], [200],
          [256, 512], [700, 3, 500, 0, 257], [33] * 20]
SIZES = [(8, 8), (136, 72), (264, 328)]


def pad_rows(counts, extra=5):
    return sum(counts) + extra


@pytest.mark.parametrize("counts", GROUPS, ids=str)
@pytest.mark.parametrize("K,N", SIZES)
def test_grouped_products(counts, K, N):
    E, R = len(counts), pad_rows(counts)
    off = offsets_of(counts)
    x = randn(R, K, seed=K + R)
    x[sum(counts):] = float("nan")          # rows behind the last group are not used
    w = randn(E, K, 2 * N, seed=2, std=K ** -0.5)
    wd = randn(E, N, K, seed=3, std=N ** -0.5)
    h = sg.grouped_fused_swiglu(x, w, off, out=torch.full((R, N), 7.0, dtype=BF16, device=DEV))
    c = sg.grouped_matmul(h, wd, off, out=torch.full((R, K), 7.0, dtype=BF16, device=DEV))
    t = sg.grouped_matmul(x, wd, off, transpose_b=True,
                          out=torch.full((R, N), 7.0, dtype=BF16, device=DEV))
    c32 = sg.grouped_matmul(h, wd, off, out_dtype=torch.float32,
                            out=torch.full((R, K), 7.0, device=DEV))
    t32 = sg.grouped_matmul(x, wd, off, transpose_b=True, out_dtype=torch.float32,
                            out=torch.full((R, N), 7.0, device=DEV))
    for v in (h, c, t, c32, t32):
        assert (v[sum(counts):] == 7.0).all()
    assert torch.equal(c32.to(BF16)[:sum(counts)], c[:sum(counts)])
    assert torch.equal(t32.to(BF16)[:sum(counts)], t[:sum(counts)])
    lo = 0
    for e, n in enumerate(counts):
        s = slice(lo, lo + n)
        want, bound, *_ = ref.swiglu(x[s], w[e])
        ref.assert_within(h[s], want, ref.rounded(want, bound), f"h of expert {e}")
        want, bound = ref.product(h[s], wd[e])
        ref.assert_within(c[s], want, ref.rounded(want, bound), f"product of expert {e}")
        ref.assert_within(c32[s], want, bound + ref.TINY, f"fp32 product of expert {e}")
        want, bound = ref.product(x[s], wd[e].t())
        ref.assert_within(t[s], want, ref.rounded(want, bound), f"transposed, expert {e}")
        lo += n


@pytest.mark.parametrize("counts", GROUPS + [[63, 64, 65, 1, 0, 2]], ids=str)
@pytest.mark.parametrize("M,N", [(8, 8), (136, 72), (264, 328)])
def test_grouped_weight_grad(counts, M, N):
    E, R = len(counts), pad_rows(counts)
    off = offsets_of(counts)
    a, g = randn(R, M, seed=M), randn(R, N, seed=N)
    a[sum(counts):] = float("nan")
    g[sum(counts):] = float("inf")
    got = sg.grouped_weight_grad(a, g, off)
    lo = 0
    for e, n in enumerate(counts):
        s = slice(lo, lo + n)
        if n == 0:
            assert not got[e].any(), f"expert {e} has no rows"
        else:
            want, bound = ref.product(a[s].t(), g[s])
            ref.assert_within(got[e], want, ref.rounded(want, bound), f"expert {e}")
        lo += n


def test_a_group_does_not_see_its_neighbours():
    """NaN and infinities in one expert's rows stay with that expert."""
    counts = [37, 100, 300]
    off = offsets_of(counts)
    R, K, N = sum(counts), 136, 72
    x, g = randn(R, K, seed=1), randn(R, N, seed=2)
    w = randn(3, K, 2 * N, seed=3)
    clean = [sg.grouped_fused_swiglu(x, w, off), sg.grouped_weight_grad(x, g, off)]
    x[37:137:3] = float("nan")
    g[38:137:5] = float("inf")
    w[1, 5] = float("nan")
    h, c = sg.grouped_fused_swiglu(x, w, off), sg.grouped_weight_grad(x, g, off)
    assert torch.equal(h[:37], clean[0][:37]) and torch.equal(h[137:], clean[0][137:])
    assert torch.equal(c[0], clean[1][0]) and torch.equal(c[2], clean[1][2])
    assert torch.isnan(h[37:137]).all() and not torch.isfinite(c[1]).any()


def test_strided_operands_and_guards():
    counts = [40, 0, 21]
    off = offsets_of(counts)
    R, K, N, E = 61, 72, 136, 3
    xw = randn(R, K + 24, seed=1)
    ww = randn(E, K + 2, 2 * N + 8, seed=2, std=0.1)
    x, w = xw[:, 8:K + 8], ww[:, :K, :2 * N]
    buf = torch.full((R + 2, N + 16), 7.0, dtype=BF16, device=DEV)
    h = sg.grouped_fused_swiglu(x, w, off, out=buf[1:R + 1, 8:N + 8])
    assert torch.equal(h, sg.grouped_fused_swiglu(x.contiguous(), w.contiguous(), off))
    buf[1:R + 1, 8:N + 8] = 7.0
    assert (buf == 7.0).all()
    wdt = randn(E, N + 8, K + 8, seed=3)[:, :N, :K]
    assert torch.equal(sg.grouped_matmul(x, wdt, off, transpose_b=True),
                       sg.grouped_matmul(x.contiguous(), wdt.contiguous(), off, transpose_b=True))
    cb = torch.full((E, K + 2, N + 16), 7.0, dtype=BF16, device=DEV)
    g = randn(R, N, seed=4)
    c = sg.grouped_weight_grad(x, g, off, out=cb[:, 1:K + 1, 8:N + 8])
    assert torch.equal(c, sg.grouped_weight_grad(x.contiguous(), g, off))
    cb[:, 1:K + 1, 8:N + 8] = 7.0
    assert (cb == 7.0).all()


def test_offsets_outside_the_rows_are_clamped():
    x, w = randn(50, 64), randn(3, 64, 128, std=0.1)
    off = torch.tensor([-5, 20, 90, 1000], dtype=torch.int32, device=DEV)
    h = sg.grouped_fused_swiglu(x, w, off, out=torch.zeros(50, 64, dtype=BF16, device=DEV))
    same = torch.tensor([0, 20, 50, 50], dtype=torch.int32, device=DEV)
    assert torch.equal(h, sg.grouped_fused_swiglu(x, w, same))


def test_many_experts_and_large_groups_are_deterministic():
    E, T, k, D, N = 1024, 700, 4, 64, 64
    ids = make_ids(T, k, E, 3, 0.0)
    order = sg.expert_order(ids, E)
    x, w = randn(T, D), randn(E, D, 2 * N, std=0.1)
    xs = sg.expert_dispatch(x, order)
    h = sg.grouped_fused_swiglu(xs, w, order.offsets)
    off = order.offsets.tolist()
    for e in (0, 17, 511, 1023):
        s = slice(off[e], off[e + 1])
        want, bound, *_ = ref.swiglu(xs[s], w[e])
        ref.assert_within(h[s], want, ref.rounded(want, bound), f"expert {e}")
    g = sg.grouped_weight_grad(xs, h, order.offsets)
    for _ in range(3):
        assert torch.equal(h, sg.grouped_fused_swiglu(xs, w, order.offsets))
        assert torch.equal(g, sg.grouped_weight_grad(xs, h, order.offsets))


# ---------------------------------------------------------------- saved pre-activations


@pytest.mark.parametrize("counts", [[1], [40, 0, 21], [300, 500], [33, 1, 700]], ids=str)
@pytest.mark.parametrize("K,N", [(8, 8), (136, 72), (64, 264)])
@pytest.mark.parametrize("checkpoint", ["bf16", "e4m3"])
def test_saved_preactivations(counts, K, N, checkpoint):
    E, R = len(counts), sum(counts)
    off = offsets_of(counts)
    x, w = randn(R, K, seed=K), randn(E, K, 2 * N, seed=N, std=K ** -0.5)
    h, pre = sg.grouped_fused_swiglu_save(x, w, off, checkpoint=checkpoint)
    assert torch.equal(h, sg.grouped_fused_swiglu(x, w, off))
    up, gate = ref.saved_values(pre)
    lo = 0
    for e, n in enumerate(counts):
        s = slice(lo, lo + n)
        _, _, u, du, g, dg = ref.swiglu(x[s], w[e])
        for got, want, bound in ((up[s], u, du), (gate[s], g, dg)):
            if checkpoint == "bf16":
                tol = ref.rounded(want, bound)
            else:
                # the block's scale is at most 2^-7 of its maximum (448 = 1.75 * 2^8, so the
                # smallest power of two is below 2 / 448 of it)
                top = torch.nn.functional.pad((want.abs() + bound), (0, -N % 32))
                top = top.unflatten(1, (-1, 32)).amax(-1, keepdim=True).expand(-1, -1, 32)
                top = top.flatten(1)[:, :N]
                tol = bound + ref.E4M3_HALF * (want.abs() + bound) + 2.0 ** -10 * top / 224
            ref.assert_within(got, want, tol, f"{checkpoint} expert {e}")
        lo += n


def exact_preact(values, rows_first=True):
    """x, w whose product is `values` exactly: one-hot rows."""
    n = values.shape[0]
    K = (n + 7) // 8 * 8
    x = torch.zeros(n, K, dtype=BF16, device=DEV)
    x[torch.arange(n), torch.arange(n)] = 1
    w = torch.zeros(K, values.shape[1], dtype=BF16, device=DEV)
    w[:n] = values
    return x, w


@pytest.mark.parametrize("N", [8, 32, 40, 136])
def test_8bit_codes_of_known_values(N):
    """Pre-activations that are known exactly give exactly the definition's codes and scales."""
    g = torch.Generator().manual_seed(N)
    v = torch.randn(64, 2 * N, generator=g)
    v *= torch.exp2(torch.randint(-60, 60, (64, 1), generator=g).float())
    v[0] = 0
    v[1] = 448.0
    v[2] = 450.0                       # just above a power-of-two border: 448 < 450 <= 896
    v[3] = torch.linspace(-1, 1, 2 * N)
    v[4] = 2.0 ** -133                 # below the smallest scale
    v[5, ::2] = 3.0e38
    v[6] = torch.where(torch.arange(2 * N) % 3 == 0, 1.0, 2.0 ** -20)
    v = v.to(BF16)
    x, w = exact_preact(v.to(DEV))
    _, pre = sg.matmul_fused_swiglu_save_preact(x, w)
    assert pre.bits == 8 and pre.hidden == N
    for half in (0, 1):
        codes, scales = ref.block_codes(v[:, half * N:(half + 1) * N].float())
        nb = scales.shape[1]
        assert torch.equal(pre.scales[:, half, :nb].cpu(), scales)
        got = pre.data[:, half, :N].cpu()
        # +0 and -0 are the same value
        got = torch.where(got == 0x80, torch.zeros_like(got), got)
        want = torch.where(codes == 0x80, torch.zeros_like(codes), codes)[:, :N]
        assert torch.equal(got, want)


def test_8bit_block_with_infinity_or_nan_reads_as_nan():
    N = 72
    v = torch.ones(8, 2 * N, dtype=BF16)
    v[1, 3] = float("nan")
    v[2, 40] = float("inf")
    v[3, N + 70] = float("-inf")
    # each row by its own expert, so that 0 * inf of the one-hot rows stays out of the others
    x = torch.zeros(8, 8, dtype=BF16, device=DEV)
    x[:, 0] = 1
    w = torch.zeros(8, 8, 2 * N, dtype=BF16, device=DEV)
    w[:, 0] = v.to(DEV)
    off = torch.arange(9, dtype=torch.int32, device=DEV)
    _, pre = sg.grouped_fused_swiglu_save(x, w, off, checkpoint="e4m3")
    up, gate = ref.saved_values(pre)
    want_up, want_gate = torch.ones(8, N), torch.ones(8, N)
    want_up[1, :32] = float("nan")
    want_up[2, 32:64] = float("nan")
    want_gate[3, 64:] = float("nan")
    assert torch.equal(torch.isnan(up.cpu()), torch.isnan(want_up))
    assert torch.equal(torch.isnan(gate.cpu()), torch.isnan(want_gate))
    grad = sg.swiglu_grad_preact_saved(torch.ones(8, N, dtype=BF16, device=DEV), pre)
    bad = torch.isnan(want_up) | torch.isnan(want_gate)
    assert torch.isnan(grad[:, N:].cpu()[bad]).all()
    assert torch.isfinite(grad[:, :N].cpu()[~bad]).all()


@pytest.mark.parametrize("R,N,end", [(1, 8, None), (37, 72, 20), (300, 264, None), (64, 136, 0),
                                     (129, 1032, 128)])
@pytest.mark.parametrize("checkpoint", ["bf16", "e4m3"])
def test_grad_preact_from_saved(R, N, end, checkpoint):
    x, w = randn(R, 64, seed=R), randn(64, 2 * N, seed=N, std=0.3)
    dy = randn(R, N, seed=9)
    _, pre = sg.matmul_fused_swiglu_save_preact(x, w, checkpoint=checkpoint)
    up, gate = ref.saved_values(pre)
    off = None
    if end is not None:
        off = torch.tensor([0, end], dtype=torch.int32, device=DEV)
    wide = torch.full((R + 2, 2 * N + 16), 7.0, dtype=BF16, device=DEV)
    out = wide[1:R + 1, 8:2 * N + 8]
    got, h = sg.swiglu_grad_preact_saved(dy, pre, offsets=off, return_h=True, out=out)
    n = R if end is None else end
    d = dy.double()
    # silu' = sig + silu * (1 - sig) cancels for negative gates: its error is relative to
    # sig * (1 + |gate|), as each of the two terms is
    sig = torch.sigmoid(gate)
    want_u, want_g = d * ref.silu(gate), d * up * ref.silu_grad(gate)
    ref.assert_within(got[:n, :N], want_u[:n],
                      ref.rounded(want_u, ref.ACT * want_u.abs())[:n], "grad up")
    err = 4 * ref.ACT * (d * up).abs() * sig * (1 + gate.abs())
    ref.assert_within(got[:n, N:], want_g[:n], ref.rounded(want_g, err)[:n], "grad gate")
    want_h = up * ref.silu(gate)
    ref.assert_within(h[:n], want_h[:n], ref.rounded(want_h, ref.ACT * want_h.abs())[:n], "h")
    out[:n] = 7.0
    assert (wide == 7.0).all()


@pytest.mark.parametrize("T,k,E,D,N,drop", [(1, 1, 1, 8, 8, 0.0), (5, 3, 4, 136, 72, 0.4),
                                            (200, 2, 4, 264, 328, 0.1), (700, 4, 7, 136, 200, 0.0),
                                            (300, 2, 2, 72, 264, 0.1), (64, 2, 4, 64, 40, 1.0)])
@pytest.mark.parametrize("checkpoint", ["bf16", "e4m3"])
@pytest.mark.parametrize("wdtype", [torch.float32, BF16, None])
def test_grouped_grad_preact(T, k, E, D, N, drop, checkpoint, wdtype):
    order = sg.expert_order(make_ids(T, k, E, T + N, drop), E)
    R, kept = T * k, int(order.offsets[-1])
    g = torch.Generator().manual_seed(T)
    rw = None if wdtype is None else torch.randn(T, 2 * k, generator=g).to(wdtype).to(DEV)[:, :k]
    xs, w = randn(R, D, seed=1), randn(E, D, 2 * N, seed=2, std=D ** -0.5)
    wd, dy = randn(E, N, D, seed=3, std=N ** -0.5), randn(R, D, seed=4)
    _, pre = sg.grouped_fused_swiglu_save(xs, w, order.offsets, checkpoint=checkpoint)
    dy[kept:] = float("nan")
    wide = torch.full((R + 2, 2 * N + 16), 7.0, dtype=BF16, device=DEV)
    out = wide[1:R + 1, 8:2 * N + 8]
    got, h = sg.grouped_grad_preact(dy, wd, pre, order, rw, out=out)
    up, gate = ref.saved_values(pre)
    off = order.offsets.tolist()
    for e in range(E):
        s = slice(off[e], off[e + 1])
        slot = order.slots[s].long()
        r = 1.0 if rw is None else rw.double()[slot // k, slot % k][:, None]
        t, dt = ref.product(dy[s], wd[e].t())
        u, ga = up[s], gate[s]
        # (the weight costs one rounding to fp32, within ACT beside the others)
        ra = abs(r) if rw is None else r.abs()
        want = r * t * ref.silu(ga)
        bound = ra * dt * ref.silu(ga).abs() + 2 * ref.ACT * want.abs()
        ref.assert_within(got[s, :N], want, ref.rounded(want, bound * 1.001), f"up, expert {e}")
        want = r * t * u * ref.silu_grad(ga)
        sig = torch.sigmoid(ga)
        bound = (ra * dt * (u * ref.silu_grad(ga)).abs()
                 + 4 * ref.ACT * ra * (t * u).abs() * sig * (1 + ga.abs()))
        ref.assert_within(got[s, N:], want, ref.rounded(want, bound * 1.001), f"gate, expert {e}")
        want = r * u * ref.silu(ga)
        ref.assert_within(h[s], want, ref.rounded(want, 2 * ref.ACT * want.abs()), f"h, expert {e}")
    out[:kept] = 7.0
    assert (wide == 7.0).all()


# ---------------------------------------------------------------- the layer


def layer_inputs(T, k, E, D, N, seed, drop=0.1, wdtype=torch.float32, D_out=None):
    D_out = D_out or D
    ids = make_ids(T, k, E, seed, drop)
    g = torch.Generator().manual_seed(seed)
    rw = torch.rand(T, k, generator=g).to(wdtype).to(DEV)
    return (randn(T, D, seed=seed), ids, rw, randn(E, D, 2 * N, seed=seed + 1, std=D ** -0.5),
            randn(E, N, D_out, seed=seed + 2, std=N ** -0.5))


def layer_reference(x, ids, rw, w, wd):
    """y in 64 bits and the bound on the kernels' result: h is rounded to bf16 on the way."""
    T, k = ids.shape
    y = torch.zeros(T, wd.shape[2], dtype=torch.float64, device=x.device)
    bound = torch.zeros_like(y)
    mag = torch.zeros_like(y)
    for e in range(w.shape[0]):
        t, j = (ids == e).nonzero(as_tuple=True)
        if t.numel() == 0:
            continue
        h, dh, *_ = ref.swiglu(x[t], w[e])
        dh = ref.rounded(h, dh)
        wde = wd[e].double()
        ye = h @ wde
        dye = dh @ wde.abs() + wd.shape[1] * ref.ACC * ((h.abs() + dh) @ wde.abs())
        r = rw[t, j].double()[:, None]
        y.index_add_(0, t, r * ye)
        bound.index_add_(0, t, r.abs() * dye)
        mag.index_add_(0, t, r.abs() * (ye.abs() + dye))
    return y, ref.rounded(y, bound + 2 * k * ref.ACC * mag)


LAYERS = [(1, 1, 1, 8, 8, None), (3, 2, 8, 72, 2440, 136), (40, 2, 4, 136, 1096, 264), (1, 2, 8, 256, 512, None), (5, 3, 4, 136, 72, None),
          (64, 8, 64, 128, 64, None), (200, 2, 4, 264, 328, 136), (1531, 4, 7, 136, 200, None)]


@pytest.mark.parametrize("T,k,E,D,N,D_out", LAYERS)
@pytest.mark.parametrize("wdtype", [torch.float32, BF16])
def test_layer_forward(T, k, E, D, N, D_out, wdtype):
    x, ids, rw, w, wd = layer_inputs(T, k, E, D, N, T, wdtype=wdtype, D_out=D_out)
    y = sg.experts_swiglu(x, ids, rw, w, wd)
    want, bound = layer_reference(x, ids, rw, w, wd)
    ref.assert_within(y, want, bound, "layer")
    # the same in separate calls (long sums over few rows are cut into ranges by the one call
    # alone, which changes the order of the additions)
    order = sg.expert_order(ids, E)
    h = sg.grouped_fused_swiglu(sg.expert_dispatch(x, order), w, order.offsets)
    ys = sg.grouped_matmul(h, wd, order.offsets, out_dtype=torch.float32)
    again = sg.expert_combine(ys, order, rw)
    if N >= 1024:
        ref.assert_within(again, want, bound, "separate calls")
    else:
        assert torch.equal(y, again)
    # in the caller's workspace, which may hold anything
    ws = torch.full((sg.experts_swiglu_workspace_bytes(T, k, E, D, N, wd.shape[2]),), 255,
                    dtype=torch.uint8, device=DEV)
    assert torch.equal(y, sg.experts_swiglu(x, ids, rw, w, wd, workspace=ws))
    if ws.numel() > 0:
        with pytest.raises(ValueError, match="workspace"):
            sg.experts_swiglu(x, ids, rw, w, wd, workspace=ws[:-256])


@pytest.mark.parametrize("T,k,E,D,N,D_out", LAYERS)
@pytest.mark.parametrize("checkpoint", ["bf16", "e4m3"])
@pytest.mark.parametrize("wdtype", [torch.float32, BF16])
def test_layer_in_training_is_its_separate_steps(T, k, E, D, N, D_out, checkpoint, wdtype):
    """The one-call forward and backward against the operators called one by one, bit for bit."""
    x, ids, rw, w, wd = layer_inputs(T, k, E, D, N, T + 3, drop=0.2, wdtype=wdtype, D_out=D_out)
    dy = randn(T, wd.shape[2], seed=4)
    y, saved = sg.experts_swiglu_save(x, ids, rw, w, wd, checkpoint=checkpoint)
    order = sg.expert_order(ids, E)
    assert torch.equal(saved.order, torch.cat([t.reshape(-1) for t in order]))
    kept = int(order.offsets[-1])
    xs = sg.expert_dispatch(x, order)
    h, pre = sg.grouped_fused_swiglu_save(xs, w, order.offsets, checkpoint=checkpoint)
    ys = sg.grouped_matmul(h, wd, order.offsets, out_dtype=torch.float32)
    assert torch.equal(saved.outputs[:kept], ys[:kept])
    for a, b in zip(ref.saved_values(saved.preact), ref.saved_values(pre)):
        assert torch.equal(a[:kept], b[:kept])
    assert torch.equal(y, sg.expert_combine(ys, order, rw))
    rows, grw = sg.expert_combine_grad(dy, ys, order, rw, weighted=False)
    gp, hw = sg.grouped_grad_preact(rows, wd, pre, order, rw)
    want = (sg.expert_combine(sg.grouped_matmul(gp, w, order.offsets, transpose_b=True,
                                                out_dtype=torch.float32), order),
            grw, sg.grouped_weight_grad(xs, gp, order.offsets),
            sg.grouped_weight_grad(hw, rows, order.offsets))
    got = sg.experts_swiglu_backward(dy, x, rw, w, wd, saved)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    for i in range(4):
        need = [j == i for j in range(4)]
        one = sg.experts_swiglu_backward(dy, x, rw, w, wd, saved, need=need)
        assert all((a is not None) == n for a, n in zip(one, need)) and torch.equal(one[i], want[i])
    none = sg.experts_swiglu_backward(dy, x, rw, w, wd, saved._replace(outputs=None),
                                      need=(True, False, True, True))
    assert none[1] is None and torch.equal(none[0], want[0])
    with pytest.raises(ValueError, match="outputs"):
        sg.experts_swiglu_backward(dy, x, rw, w, wd, saved._replace(outputs=None))


def test_training_call_refusals():
    """What does not belong together is refused before any launch."""
    x, ids, rw, w, wd = layer_inputs(4, 2, 3, 16, 24, 1, D_out=8)
    dy = randn(4, 8, seed=2)
    with pytest.raises(ValueError, match="W_down"):
        sg.experts_swiglu_save(x, ids, rw, w, wd[:2])
    saved = sg.experts_swiglu_save(x, ids, rw, w, wd)[1]
    pre = saved.preact

    def refuses(needle, kind=ValueError, g=dy, s=saved, at=x):
        with pytest.raises(kind, match=needle):
            sg.experts_swiglu_backward(g, at, rw, w, wd, s)

    refuses("SavedExperts", TypeError, s=tuple(saved))
    refuses("belong together", g=dy[:3])
    refuses("belong together", at=randn(4, 24, seed=3))
    refuses("dense", g=randn(4, 16, seed=3)[:, :8])
    refuses("saved.order", s=saved._replace(order=saved.order[:-1]))
    refuses("pre-activations", s=saved._replace(preact=pre._replace(data=pre.data[:7])))
    refuses("needed for the weights", s=saved._replace(outputs=None))
    refuses("dense fp32", s=saved._replace(outputs=saved.outputs[:7]))
    refuses("dense fp32", s=saved._replace(outputs=saved.outputs.to(BF16)))
    refuses("CUDA", at=x.cpu())


@pytest.mark.parametrize("T,k,E,D,N,D_out", LAYERS)
@pytest.mark.parametrize("checkpoint", ["bf16", "e4m3"])
def test_layer_gradients(T, k, E, D, N, D_out, checkpoint):
    """Against the formulas in 64 bits, over the pre-activations as they were kept; relative to
    the size of each gradient: two roundings to bf16 lie on the way to each result (h or the
    pre-activations' gradients, then the result), each with a root mean square below
    2^-8 / sqrt(3) of its values.  Their sum is below 2 * 2^-8."""
    x, ids, rw, w, wd = layer_inputs(T, k, E, D, N, T + 1, wdtype=BF16, D_out=D_out)
    leaves = [t.requires_grad_(True) for t in (x, rw, w, wd)]
    y = sg.fused_swiglu_experts(x, ids, rw, w, wd, checkpoint=checkpoint)
    dy = randn(*y.shape, seed=8)
    grads = torch.autograd.grad(y, leaves, dy)
    with torch.no_grad():
        if N < 1024:
            assert torch.equal(y, sg.experts_swiglu(x, ids, rw, w, wd))
        order = sg.expert_order(ids, E)
        xs = sg.expert_dispatch(x, order)
        _, pre = sg.grouped_fused_swiglu_save(xs, w, order.offsets, checkpoint=checkpoint)
        up, gate = ref.saved_values(pre)
        off = order.offsets.tolist()
        gx = torch.zeros(T, D, dtype=torch.float64, device=DEV)
        grw = torch.zeros(T, k, dtype=torch.float64, device=DEV)
        gw, gwd = torch.zeros_like(w, dtype=torch.float64), torch.zeros_like(wd, dtype=torch.float64)
        for e in range(E):
            s = slice(off[e], off[e + 1])
            slot = order.slots[s].long()
            t, j = slot // k, slot % k
            we, wde, d = w[e].double(), wd[e].double(), dy[t].double()
            h = ref.swiglu(x[t], w[e])[0]
            grw[t, j] = (d * (h @ wde)).sum(1)
            g = d * rw[t, j].double()[:, None]
            u, ga = up[s], gate[s]
            gwd[e] = (u * ref.silu(ga)).t() @ g
            gh = g @ wde.t()
            gp = torch.cat([gh * ref.silu(ga), gh * u * ref.silu_grad(ga)], 1)
            gw[e] = x[t].double().t() @ gp
            gx.index_add_(0, t, gp @ we.t())
    for got, want, name in zip(grads, (gx, grw, gw, gwd), ("x", "weights", "w", "w_down")):
        off_by = (got.double() - want).norm().item()
        assert off_by <= 2 * ref.BF16_HALF * want.norm().item() + 1e-30, (name, off_by)


def test_layer_gradients_against_differences():
    """Directional derivatives of the 64-bit layer, by central differences."""
    T, k, E, D, N = 24, 2, 3, 16, 24
    x, ids, rw, w, wd = layer_inputs(T, k, E, D, N, 5, wdtype=torch.float32)
    leaves = [t.requires_grad_(True) for t in (x, rw, w, wd)]
    y = sg.fused_swiglu_experts(x, ids, rw, w, wd)
    dy = randn(*y.shape, seed=8)
    grads = torch.autograd.grad(y, leaves, dy)

    def loss(*args):
        a, r, b, c = args
        total = 0.0
        for e in range(E):
            t, j = (ids == e).nonzero(as_tuple=True)
            up, gate = (a[t] @ b[e]).split(N, dim=1)
            ye = (up * ref.silu(gate)) @ c[e]
            total += (ye * r[t, j][:, None] * dy[t].double()).sum().item()
        return total

    base = [t.detach().double() for t in leaves]
    for i, grad in enumerate(grads):
        direction = torch.randn(base[i].shape, generator=torch.Generator().manual_seed(i),
                                dtype=torch.float64).to(DEV)
        step = 1e-4
        plus, minus = list(base), list(base)
        plus[i] = base[i] + step * direction
        minus[i] = base[i] - step * direction
        slope = (loss(*plus) - loss(*minus)) / (2 * step)
        got = (grad.double() * direction).sum().item()
        # each element of the gradient is off by at most a few bf16 half steps of the gradient's
        # size: in a random direction the errors add up like its norm
        assert abs(got - slope) <= 8 * ref.BF16_HALF * grad.double().norm().item(), i


@pytest.mark.parametrize("M,K,N", [(1, 8, 8), (7, 72, 136), (200, 136, 264), (333, 264, 72), (300, 512, 384),
                                   (1024, 256, 72)])
@pytest.mark.parametrize("checkpoint", ["bf16", "e4m3"])
def test_dense_stage_over_a_checkpoint(M, K, N, checkpoint):
    x = randn(M, K, seed=M).requires_grad_(True)
    w = randn(K, 2 * N, seed=N, std=K ** -0.5).requires_grad_(True)
    dy = randn(M, N, seed=3)
    h = sg.fused_swiglu(x, w, checkpoint=checkpoint)
    want, bound, *_ = ref.swiglu(x.detach(), w.detach())
    ref.assert_within(h.detach(), want, ref.rounded(want, bound), "h")
    gx, gw = torch.autograd.grad(h, (x, w), dy, retain_graph=True)
    with torch.no_grad():
        _, pre = sg.matmul_fused_swiglu_save_preact(x, w, checkpoint=checkpoint)
        up, gate = ref.saved_values(pre)
        gp = torch.cat([dy.double() * ref.silu(gate), dy.double() * up * ref.silu_grad(gate)], 1)
        for got, want in ((gx, gp @ w.double().t()), (gw, x.double().t() @ gp)):
            # two roundings: grad_preact and the result
            assert (got.double() - want).norm() <= 2 * ref.BF16_HALF * want.norm()
    # in its separate steps, bit for bit; one gradient alone; strided operands
    with torch.no_grad():
        gp16 = sg.swiglu_grad_preact_saved(dy, pre)
        assert torch.equal(gx, sg.matmul_bf16(gp16, w, transpose_b=True))
        assert torch.equal(gw, sg.matmul_bf16(x, gp16, transpose_a=True))
        only, none = sg.fused_swiglu_backward_saved(x, w, dy, pre, need_w=False)
        assert none is None and torch.equal(only, gx)
        none, only = sg.fused_swiglu_backward_saved(x, w, dy, pre, need_x=False)
        assert none is None and torch.equal(only, gw)
        wide = [torch.zeros(t.shape[0], t.shape[1] + 8, dtype=BF16, device=DEV)[:, :t.shape[1]]
                for t in (x, w, dy)]
        for dst, src in zip(wide, (x, w, dy)):
            dst.copy_(src)
        again = sg.fused_swiglu_backward_saved(*wide, pre)
        assert torch.equal(again[0], gx) and torch.equal(again[1], gw)
    # the checkpoint survives its backward: a second one over the same graph is the same
    again = torch.autograd.grad(h, (x, w), dy)
    assert torch.equal(again[0], gx) and torch.equal(again[1], gw)


def test_some_leaves_without_gradients():
    x, ids, rw, w, wd = layer_inputs(30, 2, 4, 64, 72, 3)
    every = [t.clone().requires_grad_(True) for t in (x, rw, w, wd)]
    dy = randn(30, 64, seed=2)
    want = torch.autograd.grad(
        sg.fused_swiglu_experts(every[0], ids, every[1], every[2], every[3]), every, dy)
    for i in range(4):
        args = [x, rw, w, wd]
        args[i] = args[i].clone().requires_grad_(True)
        y = sg.fused_swiglu_experts(args[0], ids, args[1], args[2], args[3], checkpoint="bf16")
        y.backward(dy)
        assert torch.equal(args[i].grad, want[i])
    y = sg.fused_swiglu_experts(*[t if i != 1 else ids for i, t in
                                  enumerate([every[0], None])], *every[1:])
    y.sum().backward()                      # a broadcast gradient (stride 0)
    assert all(t.grad is not None and torch.isfinite(t.grad).all() for t in every)


def test_gradients_that_start_anywhere_and_second_derivatives():
    x, ids, rw, w, wd = layer_inputs(30, 2, 4, 64, 72, 3)
    leaves = [t.requires_grad_(True) for t in (x, rw, w, wd)]
    flat = randn(30 * 64 + 3, seed=2)
    dy = flat[3:].view(30, 64)                     # contiguous, not 16-byte aligned
    assert dy.data_ptr() % 16
    got = torch.autograd.grad(sg.fused_swiglu_experts(x, ids, rw, w, wd), leaves, dy)
    want = torch.autograd.grad(sg.fused_swiglu_experts(x, ids, rw, w, wd), leaves, dy.clone())
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    xs, ws = randn(40, 64).requires_grad_(True), randn(64, 144, std=0.1).requires_grad_(True)
    flat = randn(40 * 72 + 1, seed=5)
    h = sg.fused_swiglu(xs, ws, checkpoint="e4m3")
    a = torch.autograd.grad(h, (xs, ws), flat[1:].view(40, 72), retain_graph=True)
    b = torch.autograd.grad(h, (xs, ws), flat[1:].view(40, 72).clone())
    assert all(torch.equal(u, v) for u, v in zip(a, b))
    # no second derivatives: an error, not a zero
    for out, leaf in ((sg.fused_swiglu(xs, ws, checkpoint="bf16"), xs),
                      (sg.fused_swiglu_experts(x, ids, rw, w, wd), x)):
        g, = torch.autograd.grad(out.float().square().sum(), leaf, create_graph=True)
        with pytest.raises(RuntimeError, match="once_differentiable"):
            g.float().sum().backward()


def test_module_runs_and_trains():
    torch.manual_seed(0)
    B, S, D, N, E, k = 3, 17, 64, 72, 4, 2
    for checkpoint in ("bf16", "e4m3"):
        mod = sg.PackedSwiGLUExperts(D, N, E, checkpoint=checkpoint, device=DEV)
        gate_up = torch.nn.Linear(D, 2 * N, bias=False, dtype=BF16, device=DEV)
        down = torch.nn.Linear(N, D, bias=False, dtype=BF16, device=DEV)
        mod.load_expert_(1, gate_up.weight, down.weight)
        x = randn(B, S, D, seed=1)
        ids = make_ids(B * S, k, E, 1, 0.0).view(B, S, k)
        rw = torch.rand(B, S, k, device=DEV)
        with torch.no_grad():
            y = mod(x, ids, rw)
        y2 = mod(x, ids, rw)
        assert y.shape == (B, S, D) and torch.equal(y, y2.detach())
        y2.float().square().mean().backward()
        assert mod.weight.grad.shape == mod.weight.shape and mod.weight_down.grad is not None
        lone = torch.ones_like(ids[..., :1])
        one = mod(x, lone, torch.ones(B, S, 1, device=DEV)).detach().reshape(-1, D)
        want, bound = layer_reference(x.reshape(-1, D), lone.reshape(-1, 1),
                                      torch.ones(B * S, 1, device=DEV),
                                      mod.weight.detach(), mod.weight_down.detach())
        ref.assert_within(one, want, bound, "loaded expert")
        loaded = sg.PackedSwiGLUExperts(D, N, E, device=DEV)
        loaded.load_state_dict(mod.state_dict())
        with torch.no_grad():
            assert torch.equal(loaded(x, ids, rw), y)
    lin = sg.PackedSwiGLULinear(D, N, checkpoint="e4m3", device=DEV)
    x = randn(10, D, seed=4).requires_grad_(True)
    lin(x).sum().backward()
    assert torch.isfinite(x.grad).all() and torch.isfinite(lin.weight.grad).all()


def test_row_tensors_past_32_bits():
    """More than 2^31 elements in the row tensors: rows near the end of everything."""
    T, k, E, D, N = 140000, 2, 3, 8192, 64
    ids = make_ids(T, k, E, 1, 0.01, torch.int32)
    order = sg.expert_order(ids, E)
    R, kept = T * k, int(order.offsets[-1])
    assert R * D > 2 ** 31
    gen = torch.Generator(device=DEV).manual_seed(2)
    x = torch.empty(T, D, dtype=BF16, device=DEV).normal_(generator=gen)
    xs = sg.expert_dispatch(x, order)
    w, wd = randn(E, D, 2 * N, seed=3, std=D ** -0.5), randn(E, N, D, seed=4, std=N ** -0.5)
    h, pre = sg.grouped_fused_swiglu_save(xs, w, order.offsets, checkpoint="e4m3")
    ys = sg.grouped_matmul(h, wd, order.offsets)
    off = order.offsets.tolist()
    for r in (0, off[1] - 1, off[2], kept - 1):
        e = sum(r >= o for o in off[1:])
        t = int(order.slots[r]) // k
        assert torch.equal(xs[r], x[t])
        want, bound, *_ = ref.swiglu(x[t:t + 1], w[e])
        ref.assert_within(h[r:r + 1], want, ref.rounded(want, bound), f"h row {r}")
        want, bound = ref.product(h[r:r + 1], wd[e])
        ref.assert_within(ys[r:r + 1], want, ref.rounded(want, bound), f"row {r}")
    rw = torch.rand(T, k, device=DEV)
    y = sg.expert_combine(ys, order, rw)
    gys, gw = sg.expert_combine_grad(x, ys, order, rw, out=xs)
    for t in (0, T // 2, T - 1):
        rows = order.rows[t].tolist()
        want = sum((rw[t, j].double() * ys[r].double() for j, r in enumerate(rows) if r >= 0),
                   torch.zeros(D, dtype=torch.float64, device=DEV))
        ref.assert_within(y[t], want, ref.rounded(want, 4 * ref.ACC * want.abs().max()), f"y {t}")
        for j, r in enumerate(rows):
            if r >= 0:
                want = rw[t, j].double() * x[t].double()
                ref.assert_within(gys[r], want, ref.rounded(want, ref.ACC * want.abs()), "grad row")
    grad = sg.grouped_weight_grad(gys, h, order.offsets)
    s = slice(off[2], off[3])
    want = gys[s, :8].double().t() @ h[s].double()
    mag = gys[s, :8].double().abs().t() @ h[s].double().abs()
    ref.assert_within(grad[2, :8], want, ref.rounded(want, (s.stop - s.start) * ref.ACC * mag), "C")


def test_long_routing_rows_and_wide_tokens():
    """64 choices for each token, and a layer whose experts outnumber its rows."""
    x, ids, rw, w, wd = layer_inputs(9, 64, 1024, 72, 40, 5, drop=0.3)
    want, bound = layer_reference(x, ids, rw, w, wd)
    ref.assert_within(sg.experts_swiglu(x, ids, rw, w, wd), want, bound, "64 choices")
    # the same expert several times in one token: separate slots
    ids = torch.full((7, 3), 2, device=DEV)
    want, bound = layer_reference(x[:7], ids, rw[:7, :3].contiguous(), w, wd)
    got = sg.experts_swiglu(x[:7], ids, rw[:7, :3], w, wd)
    ref.assert_within(got, want, bound, "one expert three times")


# ---------------------------------------------------------------- streams and graphs


def test_side_stream_and_stream_argument():
    x, ids, rw, w, wd = layer_inputs(300, 2, 4, 264, 328, 7)
    want = sg.experts_swiglu(x, ids, rw, w, wd)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        a = sg.experts_swiglu(x, ids, rw, w, wd)
    b = sg.experts_swiglu(x, ids, rw, w, wd, stream=s)
    order = sg.expert_order(ids, 4, stream=s)
    xs = sg.expert_dispatch(x, order, stream=s)
    h = sg.grouped_fused_swiglu(xs, w, order.offsets, stream=s)
    ys = sg.grouped_matmul(h, wd, order.offsets, stream=s, out_dtype=torch.float32)
    c = sg.expert_combine(ys, order, rw, stream=s)
    s.synchronize()
    assert torch.equal(a, want) and torch.equal(b, want) and torch.equal(c, want)


def test_two_calls_at_once_and_two_graphs():
    """Two streams at once, then two captured calls with a workspace each, replayed together."""
    one, two = layer_inputs(64, 2, 4, 264, 328, 7), layer_inputs(100, 2, 4, 264, 328, 8)
    want = [sg.experts_swiglu(*a) for a in (one, two)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        got = []
        for s, a in zip(streams, (one, two)):
            with torch.cuda.stream(s):
                got.append(sg.experts_swiglu(*a))
        torch.cuda.synchronize()
        assert all(torch.equal(g, v) for g, v in zip(got, want))
    graphs, outs = [], []
    for a in (one, two):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(sg.experts_swiglu(*a))
        graphs.append(g)
    for _ in range(3):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, v) for o, v in zip(outs, want))
    # new routing in the captured inputs
    one[1].copy_(make_ids(64, 2, 4, 99))
    graphs[0].replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], sg.experts_swiglu(*one))


def test_captured_training_step():
    x, ids, rw, w, wd = layer_inputs(200, 2, 4, 136, 72, 7)
    leaves = [t.requires_grad_(True) for t in (x, rw, w, wd)]
    dy = randn(200, 136, seed=2)

    def step():
        y = sg.fused_swiglu_experts(x, ids, rw, w, wd, checkpoint="e4m3")
        return torch.autograd.grad(y, leaves, dy)

    want = step()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step()
    for t in got:
        t.zero_()
    g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two GPUs")
def test_on_a_device_that_is_not_the_current_one():
    args = [t.to("cuda:1") for t in layer_inputs(40, 2, 4, 72, 40, 5)]
    want = sg.experts_swiglu(*(t.to("cuda:0") for t in args))
    assert torch.cuda.current_device() == 0
    got = sg.experts_swiglu(*args)
    assert got.device.index == 1 and torch.equal(got.cpu(), want.cpu())
    assert torch.cuda.current_device() == 0
    with pytest.raises(ValueError, match="different devices"):
        sg.experts_swiglu(args[0].to("cuda:0"), *args[1:])


# ---------------------------------------------------------------- calls close behind one another


def routings(T, k, E):
    """Routing that differs from call to call as far as it can: all to the first expert, all to the
    last, spread evenly, drawn with drops, none kept."""
    first = torch.zeros((T, k), dtype=torch.int64, device=DEV)
    even = (torch.arange(T * k, device=DEV) % E).view(T, k)
    return [first, first + E - 1, even, make_ids(T, k, E, 11, 0.2), first - 1]


@pytest.mark.parametrize("T,k,E", [(64, 2, 12), (1100, 2, 12), (700, 4, 40)])
def test_queued_calls_see_their_own_routing_and_weights(T, k, E):
    """Layer calls queued without a pause on one workspace and one set of buffers, with the routing
    and the weights rewritten in the stream between them: each result is that of the call alone."""
    D, N = 264, 328
    x, _, rw, w0, wd0 = layer_inputs(T, k, E, D, N, T)
    weights = [(w0, wd0), (randn(E, D, 2 * N, seed=91, std=D ** -0.5),
                           randn(E, N, D, seed=92, std=N ** -0.5))]
    ids_all = routings(T, k, E)
    alone = {}
    for i, ids in enumerate(ids_all):
        for j, (w, wd) in enumerate(weights):
            alone[i, j] = sg.experts_swiglu(x, ids, rw, w, wd)
            torch.cuda.synchronize()
    ws = torch.full((sg.experts_swiglu_workspace_bytes(T, k, E, D, N, D),), 255, dtype=torch.uint8,
                    device=DEV)
    ids, w, wd = ids_all[0].clone(), w0.clone(), wd0.clone()
    order = [(n * 3 % len(ids_all), n // 2 % 2) for n in range(40)]
    got = [torch.empty_like(x) for _ in order]
    torch.cuda.synchronize()
    for (i, j), y in zip(order, got):
        ids.copy_(ids_all[i])
        w.copy_(weights[j][0])
        wd.copy_(weights[j][1])
        sg.experts_swiglu(x, ids, rw, w, wd, out=y, workspace=ws)
    torch.cuda.synchronize()
    for n, ((i, j), y) in enumerate(zip(order, got)):
        assert torch.equal(y, alone[i, j]), (n, i, j)


@pytest.mark.parametrize("checkpoint", ["bf16", "e4m3"])
def test_queued_training_steps_see_their_own_routing_and_weights(checkpoint):
    T, k, E, D, N = 1100, 2, 12, 264, 328
    x, _, rw, w0, wd0 = layer_inputs(T, k, E, D, N, 5)
    dy = randn(T, D, seed=6)
    ids_all = routings(T, k, E)

    def step(ids, w, wd):
        y, saved = sg.experts_swiglu_save(x, ids, rw, w, wd, checkpoint=checkpoint)
        return (y, *sg.experts_swiglu_backward(dy, x, rw, w, wd, saved))

    scaled = [(w0, wd0), (w0 * 0.5, wd0 * 2)]
    alone = {}
    for i, ids in enumerate(ids_all):
        for j, (w, wd) in enumerate(scaled):
            alone[i, j] = step(ids, w, wd)
            torch.cuda.synchronize()
    ids, w, wd = ids_all[0].clone(), w0.clone(), wd0.clone()
    got = []
    for n in range(20):
        i, j = n * 3 % len(ids_all), n // 2 % 2
        ids.copy_(ids_all[i])
        w.copy_(scaled[j][0])
        wd.copy_(scaled[j][1])
        got.append((i, j, step(ids, w, wd)))
    torch.cuda.synchronize()
    for n, (i, j, result) in enumerate(got):
        for name, a, b in zip(("y", "x", "weights", "w", "w_down"), result, alone[i, j]):
            assert torch.equal(a, b), (n, i, j, name)


@pytest.mark.parametrize("T,k,E", [(64, 2, 12), (1100, 2, 12)])
def test_captured_calls_see_rewritten_routing_and_weights(T, k, E):
    """Two layers in one graph, one behind the other, replayed over rewritten routing and weights
    without a pause."""
    D, N = 264, 328
    x, _, rw, w0, wd0 = layer_inputs(T, k, E, D, N, T + 1)
    ids_all = routings(T, k, E)
    other = (randn(E, D, 2 * N, seed=91, std=D ** -0.5), randn(E, N, D, seed=92, std=N ** -0.5))
    ids, w, wd = ids_all[3].clone(), w0.clone(), wd0.clone()

    def two_layers():
        return sg.experts_swiglu(sg.experts_swiglu(x, ids, rw, w, wd), ids, rw, w, wd)

    want = {}
    for i in range(len(ids_all)):
        for j, (a, b) in enumerate([(w0, wd0), other]):
            ids.copy_(ids_all[i])
            w.copy_(a)
            wd.copy_(b)
            want[i, j] = two_layers()
            torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = two_layers()
    got = []
    for n in range(20):
        i, j = n * 3 % len(ids_all), n // 2 % 2
        ids.copy_(ids_all[i])
        w.copy_((w0, other[0])[j])
        wd.copy_((wd0, other[1])[j])
        g.replay()
        got.append((i, j, y.clone()))
    torch.cuda.synchronize()
    for n, (i, j, v) in enumerate(got):
        assert torch.equal(v, want[i, j]), (n, i, j)


# ---------------------------------------------------------------- operands of other classes


@pytest.mark.parametrize("dtype", [torch.float32, BF16])
def test_rows_that_are_parameters(dtype):
    """Rows held in a tensor subclass give what the plain tensor gives."""
    T, k, E, D, N = 60, 2, 4, 72, 40
    x, ids, rw, w, wd = layer_inputs(T, k, E, D, N, 3)
    order, dy = sg.expert_order(ids, E), randn(T, D, seed=4)
    rows = randn(T * k, D, seed=5).to(dtype)
    param = torch.nn.Parameter(rows.clone())
    assert torch.equal(sg.expert_combine(param, order, rw), sg.expert_combine(rows, order, rw))
    kept = int(order.offsets[-1])
    for a, b, n in zip(sg.expert_combine_grad(dy, param, order, rw),
                       sg.expert_combine_grad(dy, rows, order, rw), (kept, T)):
        assert torch.equal(a[:n], b[:n])
    _, saved = sg.experts_swiglu_save(x, ids, rw, w, wd)
    held = saved._replace(outputs=torch.nn.Parameter(saved.outputs.clone()))
    for a, b in zip(sg.experts_swiglu_backward(dy, x, rw, w, wd, held),
                    sg.experts_swiglu_backward(dy, x, rw, w, wd, saved)):
        assert torch.equal(a, b)


def test_weight_gradients_close_behind_one_another():
    """Results whose rows lie between the next expert's: as near as they may come, nothing shared."""
    counts, M, N, ldc = [40, 0, 21, 130], 16, 72, 160
    R, E, stride = sum(counts), len(counts), 15 * 160 + 72
    a, g = randn(R, M, seed=1), randn(R, N, seed=2)
    want = sg.grouped_weight_grad(a, g, offsets_of(counts))
    buf = torch.full((E * stride + 64,), 7.0, dtype=BF16, device=DEV)
    out = buf.as_strided((E, M, N), (stride, ldc, 1))
    assert torch.equal(sg.grouped_weight_grad(a, g, offsets_of(counts), out=out), want)
    out.fill_(7.0)
    assert (buf == 7.0).all()
    with pytest.raises(ValueError, match="overlap"):
        sg.grouped_weight_grad(a, g, offsets_of(counts),
                               out=buf.as_strided((E, M, N), (stride - 8, ldc, 1)))
