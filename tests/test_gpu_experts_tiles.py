"""The product kernel where a CTA, or a pair of them, works off several tiles.

The shapes are the smallest that reach, on a GPU of 148 SMs, what prompt-sized batches run on: tiles
of one CTA with the full 256-column accumulator, and CTA pairs with three or four tiles each (both
accumulator stages, their hand-back to the MMA issuer, a ring that goes on from tile to tile).
Tolerances are derived in ``experts_reference``."""
import pytest
import torch

import experts_reference as ref
import swiglu_fused_b200 as sg
from swiglu_fused_b200 import _lib

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16 = torch.bfloat16

# single CTAs: fewer than 256 rows per expert on average, some experts with far more or none;
# pairs: 256 and more.  The rows behind the last group belong to nobody.
UNEVEN = [700, 0, 1, 129, 40, 0, 500, 255, 300, 33] * 4
LARGE = [2100, 1, 4000]
GROUPS = {"single": (UNEVEN, 1032), "pairs": (LARGE, 2312)}
EXTRA = 37


@pytest.fixture(autouse=True)
def _device_status_clean():
    yield
    torch.cuda.synchronize()
    _lib.device_status()


def randn(*shape, seed=0, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * std).to(BF16).to(DEV)


def shuffled_order(counts):
    """One choice per token; the experts' rows as in `counts`, EXTRA tokens dropped."""
    ids = torch.cat([torch.full((n,), e) for e, n in enumerate(counts)] + [torch.full((EXTRA,), -1)])
    ids = ids[torch.randperm(ids.numel(), generator=torch.Generator().manual_seed(1))]
    return sg.expert_order(ids[:, None].to(DEV), len(counts))


def groups(counts):
    lo = 0
    for e, n in enumerate(counts):
        if n:
            yield e, slice(lo, lo + n)
        lo += n


@pytest.mark.parametrize("which", GROUPS)
@pytest.mark.parametrize("K", [72, 264])
def test_gate_up_forms(which, K):
    counts, N = GROUPS[which]
    E, R = len(counts), sum(counts) + EXTRA
    off = shuffled_order(counts).offsets
    x, w = randn(R, K, seed=K), randn(E, K, 2 * N, seed=2, std=K ** -0.5)
    x[sum(counts):] = float("nan")
    h = sg.grouped_fused_swiglu(x, w, off, out=torch.full((R, N), 7.0, dtype=BF16, device=DEV))
    saved = {}
    for checkpoint in ("bf16", "e4m3"):
        out = torch.full((R, N), 7.0, dtype=BF16, device=DEV)
        again, pre = sg.grouped_fused_swiglu_save(x, w, off, checkpoint=checkpoint, out=out)
        assert torch.equal(again, h)
        saved[checkpoint] = ref.saved_values(pre)
    assert (h[sum(counts):] == 7.0).all()
    for e, s in groups(counts):
        want, bound, u, du, g, dg = ref.swiglu(x[s], w[e])
        ref.assert_within(h[s], want, ref.rounded(want, bound), f"h of expert {e}")
        for i, (value, err) in enumerate(((u, du), (g, dg))):
            ref.assert_within(saved["bf16"][i][s], value, ref.rounded(value, err), f"bf16 {e}")
            # a block's scale is below 2 / 448 of its largest value; subnormal codes are off by at
            # most 2^-10 of it
            top = torch.nn.functional.pad(value.abs() + err, (0, -N % 32)).unflatten(1, (-1, 32))
            top = top.amax(-1, keepdim=True).expand(-1, -1, 32).flatten(1)[:, :N]
            tol = err + ref.E4M3_HALF * (value.abs() + err) + 2.0 ** -10 * top / 224
            ref.assert_within(saved["e4m3"][i][s], value, tol, f"e4m3 {e}")


@pytest.mark.parametrize("which", GROUPS)
@pytest.mark.parametrize("K", [72, 264])
@pytest.mark.parametrize("transpose_b", [False, True])
def test_product_forms(which, K, transpose_b):
    counts, N = GROUPS[which]
    E, R = len(counts), sum(counts) + EXTRA
    off = shuffled_order(counts).offsets
    a = randn(R, K, seed=K)
    a[sum(counts):] = float("nan")
    b = randn(E, N, K, seed=3) if transpose_b else randn(E, K, N, seed=3)
    c = sg.grouped_matmul(a, b, off, transpose_b=transpose_b,
                          out=torch.full((R, N), 7.0, dtype=BF16, device=DEV))
    c32 = sg.grouped_matmul(a, b, off, transpose_b=transpose_b, out_dtype=torch.float32,
                            out=torch.full((R, N), 7.0, device=DEV))
    kept = sum(counts)
    assert (c[kept:] == 7.0).all() and (c32[kept:] == 7.0).all()
    assert torch.equal(c32[:kept].to(BF16), c[:kept])
    for e, s in groups(counts):
        want, bound = ref.product(a[s], b[e].t() if transpose_b else b[e])
        ref.assert_within(c32[s], want, bound + ref.TINY, f"expert {e}")


@pytest.mark.parametrize("which", GROUPS)
@pytest.mark.parametrize("D", [72, 264])
@pytest.mark.parametrize("checkpoint", ["bf16", "e4m3"])
def test_backward_behind_the_down_projection(which, D, checkpoint):
    counts, N = GROUPS[which]
    E, R, kept = len(counts), sum(counts) + EXTRA, sum(counts)
    order = shuffled_order(counts)
    rw = torch.rand(R, 1, generator=torch.Generator().manual_seed(3)).to(DEV)
    x, w = randn(R, 64, seed=1), randn(E, 64, 2 * N, seed=2, std=0.125)
    dy, wd = randn(R, D, seed=4), randn(E, N, D, seed=5, std=N ** -0.5)
    _, pre = sg.grouped_fused_swiglu_save(x, w, order.offsets, checkpoint=checkpoint)
    dy[kept:] = float("nan")
    g, h = sg.grouped_grad_preact(dy, wd, pre, order, rw,
                                  out=torch.full((R, 2 * N), 7.0, dtype=BF16, device=DEV))
    assert (g[kept:] == 7.0).all()
    up, gate = ref.saved_values(pre)
    for e, s in groups(counts):
        r = rw.double()[order.slots[s].long()]
        t, dt = ref.product(dy[s], wd[e].t())
        u, ga = up[s], gate[s]
        want = r * t * ref.silu(ga)
        bound = r * dt * ref.silu(ga).abs() + 2 * ref.ACT * want.abs()
        ref.assert_within(g[s, :N], want, ref.rounded(want, bound * 1.001), f"up, expert {e}")
        want = r * t * u * ref.silu_grad(ga)
        bound = (r * dt * (u * ref.silu_grad(ga)).abs()
                 + 4 * ref.ACT * r * (t * u).abs() * torch.sigmoid(ga) * (1 + ga.abs()))
        ref.assert_within(g[s, N:], want, ref.rounded(want, bound * 1.001), f"gate, expert {e}")
        want = r * u * ref.silu(ga)
        ref.assert_within(h[s], want, ref.rounded(want, 2 * ref.ACT * want.abs()), f"h, expert {e}")


@pytest.mark.parametrize("M", [128, 1032])
def test_weight_gradients_of_many_tiles(M):
    """Single CTAs up to 128 rows of a result, pairs beyond; several tiles for each."""
    counts, N = GROUPS["single"]
    E, R = len(counts), sum(counts) + EXTRA
    off = shuffled_order(counts).offsets
    a, g = randn(R, M, seed=M), randn(R, N, seed=N)
    a[sum(counts):], g[sum(counts):] = float("nan"), float("inf")
    got = sg.grouped_weight_grad(a, g, off)
    full = {e for e, _ in groups(counts)}
    for e, s in groups(counts):
        want, bound = ref.product(a[s].t(), g[s])
        ref.assert_within(got[e], want, ref.rounded(want, bound), f"expert {e}")
    assert not any(got[e].any() for e in range(E) if e not in full)
