"""The mixture-of-experts operators in the self-checking build (``-DSGL_DEBUG``): the product
kernel's copies are checked against the tensors before they are issued (a violation would be
RECORDED in the status words, nothing traps).  No launch may record one, and the results equal the
normal library's bit for bit.  Runs in a child process because a process loads one copy of the library.
"""
import os
import subprocess
import sys
import textwrap

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
pytestmark = pytest.mark.gpu

CHILD = textwrap.dedent('''
    import sys
    import torch
    import swiglu_fused_b200 as sg
    from swiglu_fused_b200 import _lib
    dev, bf16 = "cuda:0", torch.bfloat16
    out = {}

    def randn(*shape, seed, std=1.0):
        g = torch.Generator().manual_seed(seed)
        return (torch.randn(shape, generator=g) * std).to(bf16).to(dev)

    def keep(name, *tensors):
        torch.cuda.synchronize()
        _lib.device_status()              # raises if a coordinate check (or a wait) failed
        for i, t in enumerate(tensors):
            out[name + (i,)] = t.cpu()

    # one row; few rows and a long sum; single CTAs, short and with 256 columns; pairs; many experts
    for (T, k, E, D, N) in [(1, 1, 1, 8, 8), (3, 2, 8, 72, 2440), (200, 2, 4, 264, 328),
                            (1531, 4, 40, 136, 1032), (1400, 2, 3, 264, 1160), (700, 4, 1024, 64, 64)]:
        g = torch.Generator().manual_seed(T)
        ids = torch.randint(0, E, (T, k), generator=g)
        ids[torch.rand(T, k, generator=g) < 0.1] = -1
        ids = ids.to(dev)
        rw = torch.rand(T, k, generator=g).to(dev)
        x, dy = randn(T, D, seed=1), randn(T, D, seed=2)
        w, wd = randn(E, D, 2 * N, seed=3, std=D ** -0.5), randn(E, N, D, seed=4, std=N ** -0.5)
        keep((T, "infer"), sg.experts_swiglu(x, ids, rw, w, wd))
        order = sg.expert_order(ids, E)
        keep((T, "order"), *order)
        for checkpoint in ("bf16", "e4m3"):
            y, saved = sg.experts_swiglu_save(x, ids, rw, w, wd, checkpoint=checkpoint)
            grads = sg.experts_swiglu_backward(dy, x, rw, w, wd, saved)
            keep((T, checkpoint), y, *grads)
        kept = int(order.offsets[-1])
        xs = sg.expert_dispatch(x, order)
        c = sg.grouped_matmul(xs, w, order.offsets)
        t = sg.grouped_matmul(xs, wd, order.offsets, transpose_b=True)
        keep((T, "products"), c[:kept], t[:kept])
    h = sg.matmul_fused_swiglu_save_preact(x, w[0], checkpoint="e4m3")[0]
    keep((0, "dense"), h)
    torch.save(out, sys.argv[1])
    print(len(out), _lib.load()._name)
''')


def _run(lib_path, out_path):
    env = dict(os.environ)
    env["PYTHONPATH"] = ROOT + os.pathsep + env.get("PYTHONPATH", "")
    if lib_path:
        env["SWIGLU_B200_LIB"] = lib_path
    else:
        env.pop("SWIGLU_B200_LIB", None)
    proc = subprocess.run([sys.executable, "-c", CHILD, out_path], env=env, capture_output=True,
                          text=True, timeout=600)
    assert proc.returncode == 0, proc.stdout[-1500:] + proc.stderr[-3000:]
    return proc.stdout


def test_experts_in_the_debug_build(tmp_path):
    import torch

    from swiglu_fused_b200 import build

    try:
        debug_lib = build.build_debug_library()
    except (OSError, RuntimeError) as e:
        pytest.skip(f"debug library not up to date and no compiler here: {e}")
    a, b = str(tmp_path / "debug.pt"), str(tmp_path / "normal.pt")
    assert "debug" in _run(debug_lib, a)
    assert "debug" not in _run(None, b)
    da, db = torch.load(a), torch.load(b)
    assert da.keys() == db.keys() and len(da) > 80
    for key, got in da.items():
        raw = torch.int16 if got.element_size() == 2 else torch.int32
        assert torch.equal(got.view(raw), db[key].view(raw)), key
