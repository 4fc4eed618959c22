"""Refusals and host arithmetic of the mixture-of-experts operators, without a GPU."""
import ctypes as C
import os
import re

import pytest
import torch

import experts_reference as ref
import swiglu_fused_b200 as sg
from swiglu_fused_b200 import _lib, build, experts

BUF = (C.c_uint8 * 4096)()
P = (C.addressof(BUF) + 15) // 16 * 16
BF16 = torch.bfloat16


def call(fn, code, needle, *args):
    lib = _lib.load()
    assert getattr(lib, fn)(*args) == code
    assert needle in lib.sgl_last_error().decode()


@pytest.mark.parametrize("change,code,needle", [
    (dict(ids=0), -1, "ids is NULL"), (dict(ids=P + 4), -4, "8-byte"), (dict(T=0), -2, "T=0"),
    (dict(k=0), -2, "k=0"), (dict(k=65, ld=65), -2, "k=65"), (dict(E=0), -2, "E=0"),
    (dict(E=1025), -2, "E=1025"), (dict(T=2 ** 31), -2, "31 bits"), (dict(ld=1), -3, "ld_ids"),
    (dict(T=1025, bytes=4096), -1, "scratch"),
    (dict(T=1025, scratch=P, bytes=60), -10, "scratch"),
    (dict(offsets=0), -1, "offsets"), (dict(slots=P + 2), -4, "slots"), (dict(rows=0), -1, "rows")])
def test_order_refusals(change, code, needle):
    a = dict(ids=P, T=4, k=2, ld=2, E=8, offsets=P, slots=P, rows=P, scratch=0, bytes=0) | change
    call("sgl_expert_order", code, needle, a["ids"], 1, a["T"], a["k"], a["ld"], a["E"],
         a["offsets"], a["slots"], a["rows"], a["scratch"], a["bytes"], None)


def test_order_scratch():
    size = _lib.load().sgl_expert_order_scratch_bytes
    assert size(1024, 2, 1024) == 0 and experts._ONE_CTA_SLOTS == 2048
    assert size(1025, 2, 8) == 2 * 8 * 4
    assert size(2 ** 30, 1, 8) == 128 * 8 * 4          # never more than 128 CTAs
    assert size(2 ** 20, 8, 1024) == 64 * 1024 * 4     # nor a table of more than 64 Ki counts
    assert size(4, 2, 1025) == -2


@pytest.mark.parametrize("change,code,needle", [
    (dict(x=0), -1, "x is NULL"), (dict(out=P + 8), -4, "16-byte"), (dict(D=12), -2, "D=12"),
    (dict(R=0), -2, "R=0"), (dict(ldx=8), -3, "ldx"), (dict(ldo=20), -3, "ldo"),
    (dict(rows=P + 1), -4, "rows")])
def test_dispatch_refusals(change, code, needle):
    a = dict(x=P, rows=P, out=P, D=16, R=8, ldx=16, ldo=16) | change
    call("sgl_expert_dispatch", code, needle, a["x"], a["rows"], a["out"], 4, 2, a["D"], a["R"],
         a["ldx"], a["ldo"], None)


@pytest.mark.parametrize("change,code,needle", [
    (dict(inp=0), -1, "in is NULL"), (dict(w=P + 2), -4, "weights"), (dict(ldw=1), -3, "ld_w"),
    (dict(ldi=8), -3, "ld_in")])
def test_combine_refusals(change, code, needle):
    a = dict(inp=P, w=P, ldw=2, ldi=16) | change
    call("sgl_expert_combine", code, needle, a["inp"], 0, P, a["w"], 0, P, 4, 2, 16, 8, a["ldi"],
         a["ldw"], 16, None)
    a.setdefault("gw", P)
    call("sgl_expert_combine_grad", code, needle, P, a["inp"], 0, P, a["w"], 0, P, a["gw"], 4, 2, 16, 8,
         16, a["ldi"], a["ldw"], 16, None)


@pytest.mark.parametrize("change,code,needle", [
    (dict(off=0), -1, "offsets"), (dict(off=P + 2), -4, "offsets"), (dict(E=1025), -2, "E=1025"),
    (dict(R=0), -2, "R=0"), (dict(K=20), -2, "multiples of 8"), (dict(ldw=16), -3, "ldw"),
    (dict(stride=8), -3, "w_stride"), (dict(stride=516), -3, "w_stride"), (dict(h=0), -1, "h is NULL"),
    (dict(R=2 ** 31), -2, "2^31")])
def test_grouped_swiglu_refusals(change, code, needle):
    a = dict(off=P, h=P, R=10, N=16, K=16, E=2, ldx=16, ldw=32, stride=512) | change
    a["ldx"] = a["K"] if a["K"] % 8 == 0 else 24
    call("sgl_grouped_fused_swiglu", code, needle, P, P, a["off"], a["h"], a["R"], a["N"], a["K"],
         a["E"], a["ldx"], a["ldw"], a["stride"], 16, None)
    call("sgl_grouped_fused_swiglu_save", code, needle, P, P, a["off"], a["h"], P, P, 8, a["R"],
         a["N"], a["K"], a["E"], a["ldx"], a["ldw"], a["stride"], 16, None)


def test_other_refusals():
    call("sgl_grouped_fused_swiglu_save", -10, "bits=4", P, P, P, P, P, P, 4, 8, 16, 16, 2, 16, 32,
         512, 16, None)
    call("sgl_grouped_fused_swiglu_save", -1, "scales", P, P, P, P, P, 0, 8, 8, 16, 16, 2, 16, 32,
         512, 16, None)
    call("sgl_grouped_matmul", -3, "ldb", P, P, P, P, 8, 16, 32, 2, 32, 16, 512, 16, 1, 0, None)
    call("sgl_grouped_matmul", -3, "b_stride", P, P, P, P, 8, 16, 32, 2, 32, 16, 256, 16, 0, 1, None)
    def grad(code, needle, **change):
        a = dict(dy=P, slots=P, weights=P, bits=8, R=8, k=2, ldw=16, stride=256, ldr=2, ldg=32,
                 scales=P) | change
        call("sgl_grouped_grad_preact", code, needle, a["dy"], P, P, a["slots"], a["weights"], 0, P,
             a["scales"], a["bits"], P, P, a["R"], 16, 16, 2, a["k"], 16, a["ldw"], a["stride"],
             a["ldr"], a["ldg"], 16, None)

    grad(-1, "dy", dy=0)
    grad(-1, "slots", slots=0)
    grad(-1, "weights", weights=0)
    grad(-1, "scales", scales=0)
    grad(-10, "bits", bits=9)
    grad(-2, "divisor", R=9)
    grad(-3, "ldw", ldw=8)
    grad(-3, "w_stride", stride=128)
    grad(-3, "ld_weights", ldr=1)
    grad(-3, "ld_grad", ldg=16)
    call("sgl_grouped_weight_grad", -3, "c_stride", P, P, P, P, 8, 16, 16, 2, 16, 16, 16, 128, None)
    call("sgl_swiglu_grad_preact_saved", -3, "ldo", P, P, P, 8, P, None, None, 8, 16, 16, 16, 0, None)
    call("sgl_swiglu_grad_preact_saved", -4, "end", P, P, P, 8, P, None, P + 2, 8, 16, 16, 32, 0, None)
    back = [P, P, P, P, P, 8, P, P, P, 8, 16, 16, 16, 32, 16, None, None, None]

    def backward(code, needle, at, value):
        call("sgl_fused_swiglu_backward_saved", code, needle, *(back[:at] + [value] + back[at + 1:]))

    backward(-1, "x is NULL", 0, None)
    backward(-1, "dy is NULL", 2, None)
    backward(-1, "scales", 4, None)
    backward(-10, "bits", 5, 7)
    backward(-4, "grad_w", 8, P + 2)
    backward(-2, "M=0", 9, 0)
    backward(-3, "ldw", 13, 16)
    backward(-3, "lddy", 14, 8)
    call("sgl_experts_swiglu", -10, "workspace", P, P, 1, P, 0, P, P, P, P, 64, 4, 2, 8, 16, 16, 16,
         16, 2, 2, 32, 512, 16, 256, 16, None)
    n = _lib.load().sgl_experts_swiglu_workspace_bytes(4, 2, 8, 16, 16, 16)
    call("sgl_experts_swiglu", -3, "ldd", P, P, 1, P, 0, P, P, P, P, n, 4, 2, 8, 16, 16, 16,
         16, 2, 2, 32, 512, 8, 256, 16, None)
    size = _lib.load().sgl_experts_swiglu_train_workspace_bytes
    fwd, bwd = size(4, 2, 8, 16, 16, 16, 0), size(4, 2, 8, 16, 16, 16, 1)
    assert fwd >= 8 * (16 + 16) * 2 and bwd >= 8 * 32 * 2 + 8 * 16 * 4
    assert size(4, 2, 1025, 16, 16, 16, 1) == -2

    def save(code, needle, **change):
        a = dict(ids=P, order=P, scales=P, ys=P, bits=8, bytes=fwd, ldd=16, ld_ids=2) | change
        call("sgl_experts_swiglu_save", code, needle, P, a["ids"], 1, P, 0, P, P, P, a["order"], P,
             a["scales"], a["bits"], a["ys"], P, a["bytes"], 4, 2, 8, 16, 16, 16, 16, a["ld_ids"], 2,
             32, 512, a["ldd"], 256, None)

    def grads(code, needle, **change):
        a = dict(gy=P, order=P, scales=P, ys=P, gr=P, gw=P, bits=8, bytes=bwd, ldw=32) | change
        call("sgl_experts_swiglu_backward", code, needle, a["gy"], P, P, 0, P, P, a["order"], P,
             a["scales"], a["bits"], a["ys"], P, a["gr"], a["gw"], P, P, a["bytes"], 4, 2, 8, 16, 16,
             16, 16, 2, a["ldw"], 512, 16, 256, None)

    save(-1, "ids", ids=0)
    save(-1, "order", order=0)
    save(-1, "scales", scales=0)
    save(-1, "ys", ys=0)
    save(-10, "bits", bits=32)
    save(-10, "workspace", bytes=fwd - 1)
    save(-3, "ldd", ldd=8)
    save(-3, "ld_ids", ld_ids=1)
    grads(-1, "grad_y", gy=0)
    grads(-4, "order", order=P + 2)
    grads(-1, "ys", ys=0)
    grads(-4, "grad_weights", gr=P + 2)
    grads(-4, "grad_w", gw=P + 8)
    grads(-10, "bits", bits=0)
    grads(-10, "workspace", bytes=bwd - 1)
    grads(-3, "ldw", ldw=16)
    assert _lib.load().sgl_experts_swiglu_workspace_bytes(0, 2, 8, 16, 16, 16) == -2
    assert _lib.load().sgl_preact_bytes(8, 4, 12, None, None, None) == -2


def test_workspace_holds_every_part():
    T, k, E, D, N, Do = 5, 3, 7, 24, 40, 16
    n = sg.experts_swiglu_workspace_bytes(T, k, E, D, N, Do)
    assert n >= 4 * (E + 1) + 8 * T * k + 2 * T * k * (D + N + 2 * Do)
    assert n <= 4 * (E + 1) + 8 * T * k + 2 * T * k * (D + N + 2 * Do) + 6 * 256
    # few rows and a long sum: partial rows of the down projection
    one = sg.experts_swiglu_workspace_bytes(1, 2, 8, 64, 14336, 4096)
    assert one >= 2 * 2 * (64 + 14336) + 2 * 4096 * 4 * 8
    with pytest.raises(ValueError):
        sg.experts_swiglu_workspace_bytes(1, 65, E, D, N, Do)


@pytest.mark.parametrize("N,half,scale", [(8, 32, 2), (32, 32, 2), (40, 64, 2), (72, 96, 4),
                                          (14336, 14336, 448)])
def test_preact_shapes(N, half, scale):
    assert experts._preact_shapes(8, 5, N) == ((5, 2, half), (5, 2, scale))
    assert experts._preact_shapes(16, 5, N) == ((5, 2, half), None)
    pitch, scale_bytes, scale_pitch = C.c_int64(), C.c_int64(), C.c_int64()
    size = _lib.load().sgl_preact_bytes
    assert size(8, 5, N, C.byref(pitch), C.byref(scale_bytes), C.byref(scale_pitch)) == 10 * half
    assert (pitch.value, scale_bytes.value, scale_pitch.value) == (2 * half, 10 * scale, 2 * scale)
    assert size(16, 5, N, None, None, None) == 20 * half


def test_python_refusals():
    ids = torch.zeros((4, 2), dtype=torch.int64)
    with pytest.raises(ValueError, match="CUDA"):
        sg.expert_order(ids, 4)
    with pytest.raises(TypeError, match="expert_ids"):
        sg.expert_order(ids.float(), 4)
    with pytest.raises(ValueError, match="tokens, choices"):
        sg.expert_order(ids.view(-1), 4)
    with pytest.raises(ValueError, match="choices per token"):
        sg.expert_order(torch.zeros((4, 65), dtype=torch.int64), 4)
    order = sg.ExpertOrder(torch.zeros(5, dtype=torch.int32), torch.zeros(8, dtype=torch.int32),
                           torch.zeros((4, 2), dtype=torch.int32))
    x = torch.zeros((4, 16), dtype=BF16)
    with pytest.raises(ValueError, match="CUDA"):
        sg.expert_dispatch(x, order)
    with pytest.raises(TypeError, match="ExpertOrder"):
        sg.expert_combine(x, (order.offsets, order.slots, order.rows))
    w = torch.zeros((4, 16, 32), dtype=BF16)
    with pytest.raises(ValueError, match="CUDA"):
        sg.grouped_fused_swiglu(x, w, order.offsets)
    with pytest.raises(ValueError, match="checkpoint"):
        sg.fused_swiglu(x, w[0], checkpoint="int8")
    with pytest.raises(ValueError, match="checkpoint"):
        sg.PackedSwiGLUExperts(16, 16, 4, checkpoint="fp8")
    with pytest.raises(ValueError, match="multiples of 8"):
        sg.PackedSwiGLUExperts(16, 12, 4)
    with pytest.raises(TypeError, match="SavedPreact"):
        sg.swiglu_grad_preact_saved(x, x)


def test_training_call_refusals():
    """The layer's one-call forward and backward have no CPU path."""
    x, ids, rw = torch.zeros((4, 16), dtype=BF16), torch.zeros((4, 2), dtype=torch.int32), torch.zeros(4, 2)
    w, wd = torch.zeros((3, 16, 48), dtype=BF16), torch.zeros((3, 24, 8), dtype=BF16)
    with pytest.raises(ValueError, match="checkpoint"):
        sg.experts_swiglu_save(x, ids, rw, w, wd, checkpoint="int8")
    with pytest.raises(ValueError, match="CUDA"):
        sg.experts_swiglu_save(x, ids, rw, w, wd)
    pre = sg.SavedPreact(torch.zeros((8, 48), dtype=BF16), None, 16, 24)
    saved = sg.SavedExperts(torch.zeros(3 + 1 + 16, dtype=torch.int32), pre, torch.zeros(8, 8))
    with pytest.raises(ValueError, match="CUDA"):
        sg.experts_swiglu_backward(torch.zeros((4, 8), dtype=BF16), x, rw, w, wd, saved)


def test_a_bad_stream_leaves_the_current_device(monkeypatch):
    """A call whose stream is not one leaves the device current that was."""
    from swiglu_fused_b200 import experts
    at = [1]
    monkeypatch.setattr(torch.cuda, "current_device", lambda: at[-1])
    monkeypatch.setattr(torch.cuda, "set_device", at.append)
    with pytest.raises(ValueError):
        with experts._launch("no stream", torch.device("cuda", 0)):
            pass
    assert at == [1, 0, 1]


def test_module_parameters_and_expert_loading():
    mod = sg.PackedSwiGLUExperts(16, 24, 3, out_features=8)
    assert mod.weight.shape == (3, 16, 48) and mod.weight_down.shape == (3, 24, 8)
    gate_up, down = torch.randn(48, 16).to(BF16), torch.randn(8, 24).to(BF16)
    mod.load_expert_(2, gate_up, down)
    assert torch.equal(mod.weight[2].detach(), gate_up.t())
    assert torch.equal(mod.weight_down[2].detach(), down.t())
    with pytest.raises(ValueError, match="gate_up"):
        mod.load_expert_(0, gate_up.t(), down)
    assert set(mod.state_dict()) == {"weight", "weight_down"}


def test_reference_block_codes():
    """The plain form itself: smallest power of two that holds the block, nearest e4m3 value."""
    v = torch.tensor([[448.0] + [1.0] * 31, [449.0] + [0.0] * 31, [0.0] * 32])
    codes, scales = ref.block_codes(v)
    assert scales.view(-1).tolist() == [127, 128, 0]
    assert codes[0, 0].item() == 0x7e and codes[0, 1].item() == 0x38
    assert codes[1, 0].item() == 0x76              # 224.5 -> 224


def _kernels(source):
    """(name, body) of every kernel of a source file, comments taken out."""
    text = re.sub(r"//[^\n]*", "", source)
    for m in re.finditer(r"__global__ void(?:\s+__launch_bounds__\(.*?\))?\s+(\w+)\(", text):
        start = text.index("{", m.end())
        depth, end = 1, start + 1
        while depth:
            depth += {"{": 1, "}": -1}.get(text[end], 0)
            end += 1
        yield m.group(1), text[start + 1:end - 1]


@pytest.mark.parametrize("name", ["experts_order.cuh", "experts_products.cuh", "swiglu_preact.cuh"])
def test_kernels_wait_before_they_touch_memory(name):
    """These kernels are launched beside the end of the launch before them.  What that launch, or an
    earlier one, has written is visible to a kernel only behind its own griddepcontrol.wait: the wait
    is unconditional, and no global memory is read or written before it."""
    with open(os.path.join(build.CSRC_DIR, name)) as f:
        kernels = list(_kernels(f.read()))
    assert kernels
    for kernel, body in kernels:
        at = body.find("griddepcontrol.wait")
        assert at >= 0, f"{kernel} does not wait"
        before = body[:at]
        assert before.count("{") == before.count("}"), f"{kernel} waits under a condition"
        # (kernel parameters used as addresses, TMA copies, and the helpers that read global memory)
        touches = re.search(r"p\.\w+\s*\[|\*\s*p\.|tma_|\.load\(|row_lo\(|order_key\(|row_of\(|"
                            r"load_weight\(|\.run\(", before)
        assert touches is None, f"{kernel}: {touches and touches.group()!r} before the wait"


def test_rows_of_any_tensor_class():
    """fp32 rows are recognised in a tensor subclass too: what is refused here is the device alone."""
    order = sg.ExpertOrder(torch.zeros(5, dtype=torch.int32), torch.zeros(8, dtype=torch.int32),
                           torch.zeros((4, 2), dtype=torch.int32))
    for dtype in (torch.float32, BF16):
        rows = torch.nn.Parameter(torch.zeros((8, 16), dtype=dtype))
        with pytest.raises(ValueError, match="rows must be a CUDA tensor"):
            experts._rows_matrix(rows, "rows")
    with pytest.raises(TypeError, match="float64"):
        experts._rows_matrix(torch.nn.Parameter(torch.zeros((8, 16), dtype=torch.float64)), "rows")
    with pytest.raises(TypeError, match="list"):
        experts._rows_matrix([1.0], "rows")
    with pytest.raises(ValueError, match="CUDA"):
        sg.expert_combine(torch.nn.Parameter(torch.zeros((8, 16))), order)


@pytest.mark.parametrize("M,N,ldc,stride", [(16, 16, 16, 240), (16, 16, 24, 360), (16, 16, 24, 368),
                                            (8, 64, 72, 504)])
def test_weight_gradients_that_overlap_are_refused(M, N, ldc, stride):
    """The last row of one expert's result would be the first of the next one's."""
    assert stride < (M - 1) * ldc + N
    call("sgl_grouped_weight_grad", -3, "c_stride", P, P, P, P, 8, M, N, 2, M, N, ldc, stride, None)


@pytest.mark.parametrize("bits", [8, 16])
def test_preact_bytes_of_no_rows_and_of_fewer(bits):
    size = _lib.load().sgl_preact_bytes
    pitch, scale_bytes, scale_pitch = C.c_int64(-7), C.c_int64(-7), C.c_int64(-7)
    sizes = [C.byref(v) for v in (pitch, scale_bytes, scale_pitch)]
    for rows in (-1, -(2 ** 40)):
        call("sgl_preact_bytes", -2, f"rows={rows}", bits, rows, 40, *sizes)
    assert (pitch.value, scale_bytes.value, scale_pitch.value) == (-7, -7, -7)
    assert size(bits, 0, 40, *sizes) == 0
    assert (pitch.value, scale_bytes.value) == (2 * 64 * bits // 8, 0)
    assert scale_pitch.value == (4 if bits == 8 else 0)


def test_bounds_of_an_8bit_block():
    """The plain form keeps 2^-4 of a value down to 2^-13 of its block's largest, 2^-10 of the scale
    below; 2^-15 of the largest is too far down for the relative bound."""
    largest = torch.linspace(225, 448, 300)
    for shift, within in ((0, True), (7, True), (13, True), (15, False)):
        worst = 0.0
        for part in torch.linspace(1, 1.99, 31):
            v = torch.zeros(300, 32)
            v[:, 0], v[:, 1] = largest, largest * 2.0 ** -shift * part
            if shift == 0:
                v[:, 1] = largest / part
            codes, scales = ref.block_codes(v)
            assert (scales == 127).all()
            got = codes.view(torch.float8_e4m3fn).double()[:, 1]
            off = (got - v[:, 1].double()).abs()
            worst = max(worst, (off / v[:, 1].double()).max().item())
            assert (off <= torch.maximum(2.0 ** -4 * v[:, 1].double(), torch.tensor(2.0 ** -10))).all()
        assert (worst <= 2.0 ** -4) == within, (shift, worst)
    tiny = torch.full((1, 32), 2.0 ** -133)            # a scale held at 2^-127
    codes, scales = ref.block_codes(tiny)
    assert scales.item() == 0
    value = codes.view(torch.float8_e4m3fn).double()[0, 0] * 2.0 ** -127
    assert abs(value - 2.0 ** -133) <= 2.0 ** -137
