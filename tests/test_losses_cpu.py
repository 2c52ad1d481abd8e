"""What the losses refuse, and what their C entry points say of a problem, without a device."""
import ctypes

import pytest
import torch

import tensorcomprehensions_b200 as tc
from tensorcomprehensions_b200 import cabi

PTR = ctypes.c_void_p(1 << 20)  # never dereferenced: the calls fail before any work


def ce(N=100, D=64, V=1000, ldx=None, ldw=None, dtype=cabi.BF16, index_bytes=8, pack_w=0):
    return cabi.LinearCe(N, D, V, D if ldx is None else ldx, D if ldw is None else ldw, -100, dtype, index_bytes, pack_w, 0)


def workspace(p):
    f, b = ctypes.c_int64(), ctypes.c_int64()
    return cabi.lib().tcb200_linear_ce_workspace(ctypes.byref(p), ctypes.byref(f), ctypes.byref(b)), f.value, b.value


def test_workspace_follows_the_problem_and_stays_far_below_the_logits():
    st, f, b = workspace(ce())
    assert st == 0 and 0 < f < b
    # 8192 x 131072: the logits would take 2 GiB in 16 bits; the forward pass keeps 8 bytes per 128 of them
    st, f, b = workspace(ce(8192, 4096, 131072))
    assert st == 0 and f < (200 << 20) and b < (640 << 20)
    assert workspace(ce(8192, 4096, 131072, pack_w=1))[1] > f
    assert workspace(ce(100, 64, 1000, dtype=cabi.F32))[2] > workspace(ce(100, 64, 1000))[2]
    assert workspace(ce(0))[0] == 0


def test_linear_ce_argument_checks():
    for bad in (dict(N=-1), dict(D=0), dict(V=0), dict(ldx=63), dict(ldw=63), dict(dtype=3), dict(dtype=-1), dict(index_bytes=2)):
        assert workspace(ce(**bad))[0] == -1, bad
    assert workspace(ce(D=65))[0] == -4                      # rows of W off their 16-byte boundaries, not packed
    assert workspace(ce(D=65, pack_w=1))[0] == 0
    assert workspace(ce(D=65, dtype=cabi.F32))[0] == 0       # always packed
    assert workspace(ce(V=1 << 31))[0] == -7 and workspace(ce(D=1 << 21))[0] == -7
    L, p = cabi.lib(), ce()
    _, f, b = workspace(p)
    assert L.tcb200_linear_ce_workspace(None, None, None) == -1
    r = ctypes.byref(p)
    assert L.tcb200_linear_ce_forward(r, None, PTR, PTR, PTR, PTR, PTR, f, None, None) == -1
    assert L.tcb200_linear_ce_forward(r, PTR, PTR, PTR, PTR, PTR, PTR, f - 1, None, None) == -1
    assert L.tcb200_linear_ce_forward(r, PTR, PTR, PTR, PTR, PTR, ctypes.c_void_p((1 << 20) + 16), f, None, None) == -4
    assert L.tcb200_linear_ce_forward(r, PTR, ctypes.c_void_p((1 << 20) + 2), PTR, PTR, PTR, PTR, f, None, None) == -4
    assert L.tcb200_linear_ce_backward(r, PTR, PTR, PTR, PTR, PTR, -1, PTR, PTR, PTR, b, None, None) == -1
    assert L.tcb200_linear_ce_backward(r, PTR, PTR, PTR, PTR, None, 1, PTR, PTR, PTR, b, None, None) == -1
    assert L.tcb200_linear_ce_backward(r, PTR, PTR, PTR, PTR, PTR, 1, PTR, PTR, PTR, b - 1, None, None) == -1
    assert L.tcb200_linear_ce_backward(r, PTR, PTR, PTR, PTR, PTR, 1, None, None, None, 0, None, None) == 0   # nothing asked for
    assert L.tcb200_linear_ce_forward(ctypes.byref(ce(0)), None, PTR, None, None, None, None, 0, None, None) == 0


def kd(N=10, V=1000, K=8, ldl=None, ldi=None, ldt=None, temperature=1.0, dtype=cabi.BF16, teacher=cabi.BF16, index_bytes=8):
    return cabi.TopkDistill(N, V, K, V if ldl is None else ldl, K if ldi is None else ldi, K if ldt is None else ldt, temperature, dtype, teacher, index_bytes)


def test_topk_distill_argument_checks():
    L = cabi.lib()

    def call(p):
        r = ctypes.byref(p)
        # a null among the pointers: a problem that passes its own checks is refused for it, before any launch
        f = L.tcb200_topk_distill_forward(r, PTR, PTR, PTR, PTR, None, None)
        assert f == L.tcb200_topk_distill_backward(r, PTR, PTR, PTR, PTR, PTR, 1, None, None)
        return f

    assert call(kd()) == -1
    assert call(kd(N=0)) == 0
    for bad in (dict(N=-1), dict(V=0), dict(K=0), dict(ldl=999), dict(ldi=7), dict(ldt=7), dict(dtype=9), dict(teacher=-1), dict(index_bytes=1),
                dict(temperature=0.0), dict(temperature=-1.0), dict(temperature=float("inf")), dict(temperature=float("nan"))):
        assert call(kd(**{"N": 0, **bad})) == -1, bad      # N = 0 would succeed if the check let it through
    assert call(kd(N=0, K=cabi.TOPK_MAX + 1)) == -7 and call(kd(N=0, V=1 << 31)) == -7 and call(kd(N=1 << 27)) == -7
    assert L.tcb200_topk_distill_forward(None, PTR, PTR, PTR, PTR, PTR, None) == -1


def test_tensors_off_the_device_are_refused():
    x, w, t = torch.zeros(4, 8), torch.zeros(16, 8), torch.zeros(4, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="X must be a CUDA tensor"):
        tc.linear_cross_entropy(x, w, t)
    with pytest.raises(RuntimeError, match="logits must be a CUDA tensor"):
        tc.topk_distillation(torch.zeros(4, 16), torch.zeros(4, 2, dtype=torch.int64), torch.zeros(4, 2))


def test_cpp_entry_points_without_a_device():
    if torch.cuda.is_available():
        pytest.skip("covered by the gpu variant")
    from test_cpp_api import _build, _run
    r = _run(_build("losses"))
    assert r.returncode == 0, r.stdout + r.stderr
    assert "losses ok (gpu=0)" in r.stdout


@pytest.mark.gpu
def test_cpp_entry_points(cuda):
    from test_cpp_api import _build, _run
    r = _run(_build("losses"))
    assert r.returncode == 0, r.stdout + r.stderr
    assert "losses ok (gpu=1)" in r.stdout


def test_a_peers_shared_memory_is_touched_only_behind_a_cluster_barrier():
    """In every kernel source: a store into another CTA's shared memory stands behind a wait of the same kernel on its cluster's barrier,
    since a CTA that has not started has no shared memory to store into."""
    import glob
    import os
    import re
    kernels = os.path.join(os.path.dirname(cabi.__file__), "csrc", "kernels")
    stores = 0
    for path in glob.glob(os.path.join(kernels, "*.cu")) + glob.glob(os.path.join(kernels, "*.cuh")):
        text = re.sub(r"//[^\n]*", "", open(path).read())
        for body in re.split(r"\b__global__\b", text)[1:]:
            for at in (m.start() for m in re.finditer(r"\bst\.(?:async\.)?shared::cluster", body)):
                stores += 1
                assert re.search(r"\bcluster_(?:wait|sync_all)\(\)", body[:at]), path
    assert stores > 0


def _build_with_streams():
    """tests/cpp/losses_streams.cc, which makes streams with torch's C++ classes: those need the CUDA headers."""
    import os
    import subprocess
    from torch.utils import cpp_extension
    pkg = os.path.dirname(cabi.__file__)
    src, exe = os.path.join(os.path.dirname(__file__), "cpp", "losses_streams.cc"), os.path.join(pkg, "build", "losses_streams")
    os.makedirs(os.path.dirname(exe), exist_ok=True)
    if not os.path.exists(exe) or any(os.path.getmtime(f) > os.path.getmtime(exe) for f in (src, os.path.join(pkg, "libtc_core.so"))):
        tlib = os.path.join(os.path.dirname(torch.__file__), "lib")
        cmd = ["/usr/bin/g++", "-std=c++17", "-O1", "-w", "-D_GLIBCXX_USE_CXX11_ABI=%d" % int(torch._C._GLIBCXX_USE_CXX11_ABI),
               "-I" + os.path.join(os.path.dirname(pkg), "include"), "-I/usr/local/cuda/include"] + ["-I" + p for p in cpp_extension.include_paths()] + \
              [src, "-o", exe, "-L" + pkg, "-ltc_core", "-ltcb200", "-L" + tlib, "-ltorch", "-ltorch_cpu", "-lc10", "-Wl,-rpath," + pkg,
               "-Wl,-rpath," + tlib, "-Wl,--no-as-needed", "-ltorch_cuda", "-lc10_cuda", "-Wl,--as-needed", "-L/usr/local/cuda/lib64", "-lcudart"]
        r = subprocess.run(cmd, capture_output=True, text=True)
        assert r.returncode == 0, r.stderr[-3000:]
    return exe


def test_cpp_entry_points_on_named_streams_build():
    if torch.cuda.is_available():
        pytest.skip("covered by the gpu variant")
    from test_cpp_api import _run
    r = _run(_build_with_streams())
    assert r.returncode == 0, r.stdout + r.stderr
    assert "losses on streams ok (gpu=0)" in r.stdout


@pytest.mark.gpu
def test_cpp_entry_points_on_named_streams(cuda):
    from test_cpp_api import _run
    r = _run(_build_with_streams())
    assert r.returncode == 0, r.stdout + r.stderr
    assert "losses on streams ok (gpu=1)" in r.stdout


def test_tangents_are_refused():
    """Forward-mode derivatives: a dual tensor does not require grad, and its tangent must not get lost."""
    import torch.autograd.forward_ad as fwd
    x, w, t = torch.zeros(4, 8), torch.zeros(16, 8), torch.zeros(4, dtype=torch.int64)
    z, i, s = torch.zeros(4, 16), torch.zeros(4, 2, dtype=torch.int64), torch.zeros(4, 2)
    with fwd.dual_level():
        dual = lambda a: fwd.make_dual(a, torch.ones_like(a))  # noqa: E731
        for args in ((dual(x), w, t), (x, dual(w), t)):
            with pytest.raises(RuntimeError, match="linear_cross_entropy has no forward-mode derivative"):
                tc.linear_cross_entropy(*args)
            with torch.no_grad(), pytest.raises(RuntimeError, match="no forward-mode derivative"):
                tc.linear_cross_entropy(*args)
        for args in ((dual(z), i, s), (z, i, dual(s))):
            with pytest.raises(RuntimeError, match="topk_distillation has no forward-mode derivative"):
                tc.topk_distillation(*args)


def _build_gave_up():
    import os
    import subprocess
    from tensorcomprehensions_b200 import _build
    kernels, exe = os.path.join(_build.CSRC, "kernels"), os.path.join(_build.PKG, "build", "losses_gave_up")
    src = os.path.join(os.path.dirname(__file__), "cpp", "losses_gave_up.cu")
    os.makedirs(os.path.dirname(exe), exist_ok=True)
    if not os.path.exists(exe) or any(os.path.getmtime(f) > os.path.getmtime(exe) for f in (src, os.path.join(_build.PKG, "libtcb200.so"))):
        r = subprocess.run([_build._nvcc()] + _build.NVCC_FLAGS + ["-I" + _build.INCLUDE, "-I" + kernels, src, "-o", exe], capture_output=True, text=True)
        assert r.returncode == 0, r.stderr[-3000:]
    return exe


def test_gradients_behind_a_wait_that_gave_up_build():
    if torch.cuda.is_available():
        pytest.skip("covered by the gpu variant")
    from test_cpp_api import _run
    r = _run(_build_gave_up())
    assert r.returncode == 0 and "gave up ok (gpu=0)" in r.stdout, r.stdout + r.stderr


@pytest.mark.gpu
def test_gradients_behind_a_wait_that_gave_up(cuda):
    from test_cpp_api import _run
    r = _run(_build_gave_up())
    assert r.returncode == 0 and "gave up ok (gpu=1)" in r.stdout, r.stdout + r.stderr


def test_temperatures_whose_square_is_no_normal_number_are_refused():
    """At 1e-39, 1 / T is infinite and the loss NaN; at 1e-20, T^2 is lost; at 1e20 it is infinite."""
    L = cabi.lib()
    for temperature in (1e-45, 1e-39, 1e-38, 1e-20, 1.0e-19, 2.0**64, 1e20, 3e38):
        r = ctypes.byref(kd(N=0, temperature=temperature))   # N = 0 would succeed if the check let it through
        assert L.tcb200_topk_distill_forward(r, PTR, PTR, PTR, PTR, PTR, None) == -1, temperature
        assert L.tcb200_topk_distill_backward(r, PTR, PTR, PTR, PTR, PTR, 1, PTR, None) == -1, temperature
    for temperature in (2.0**-63, 1e-3, 1.0, 100.0, 1e19):
        assert L.tcb200_topk_distill_forward(ctypes.byref(kd(N=0, temperature=temperature)), PTR, PTR, PTR, PTR, PTR, None) == 0, temperature
