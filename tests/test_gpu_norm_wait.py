"""A wait for a row that runs out: the kernel says so, ends with no copy on its
way, and writes nothing but its outputs.  The kernels are compiled with waits
that give up at once (norm_wait.cu); the copies they wait for are in order."""
import ctypes as C
import os
import subprocess

import pytest
import torch

import orthossm_b200 as O
from orthossm_b200 import _lib as L
from orthossm_b200 import build

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    out = str(tmp_path_factory.mktemp("norm") / "norm_wait.so")
    subprocess.run([build.nvcc(), *build.ARCH, "-O3", "-std=c++17", "-shared", "-Xcompiler", "-fPIC", "-cudart", "shared",
                    f"-I{build.INCLUDE}", f"-I{build.CSRC}", "-o", out,
                    os.path.join(os.path.dirname(__file__), "norm_wait.cu")], check=True)
    so = C.CDLL(out)
    so.norm_wait_bytes.restype = C.c_size_t
    return so


class Buffers:
    """Outputs between guards that no kernel may touch."""

    def __init__(self):
        self.all = []

    def new(self, *shape, dtype=BF):
        n = 1
        for k in shape:
            n *= k
        whole = torch.full((n + 4096,), 7.0, dtype=dtype, device="cuda")
        self.all.append((whole, n))
        return whole[2048:2048 + n].view(shape)

    def intact(self):
        return all(bool((w[:2048] == 7).all()) and bool((w[2048 + n:] == 7).all()) for w, n in self.all)


@pytest.mark.parametrize("T,d,post", [(5000, 512, 0), (3, 512, 0), (2999, 1000, 0), (4001, 2048, 0), (2000, 512, 1),
                                      (1500, 1000, 1), (4000, 256, 1)])
def test_a_wait_that_runs_out(lib, T, d, post):
    x, y, gr, gh = (torch.randn(T, d, device="cuda").to(BF) for _ in range(4))
    w = torch.ones(d, device="cuda")
    before = O.residual_norm(x, y, w, post_norm="rms" if post else None)
    buf = Buffers()
    r, h, dx, dy = (buf.new(T, d) for _ in range(4))
    stats = buf.new(4, T, dtype=torch.float32)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    a = L.NormArgs(tokens=T, dim=d, stream_dtype=L.OSSM_BF16, dtype=L.OSSM_BF16, x=x.data_ptr(), x_stride=d, y=y.data_ptr(),
                   y_stride=d, scale=1.0, norm=L.OSSM_NORM_RMS, post_norm=post, eps=1e-6, post_eps=1e-6,
                   weight=w.data_ptr(), weight_dtype=L.OSSM_F32, r=r.data_ptr(), h=h.data_ptr(), stats=stats.data_ptr(),
                   status=status.data_ptr())
    stream = C.c_void_p(torch.cuda.current_stream().cuda_stream)
    if d > 256:
        assert lib.norm_wait_fwd(C.byref(a), stream) == 0
        torch.cuda.synchronize()
        assert status.item() == L.OSSM_ETIMEOUT and buf.intact()
        status.zero_()
    a.r = None
    a.grad_r, a.grad_h, a.grad_r_stride, a.grad_h_stride = gr.data_ptr(), gh.data_ptr(), d, d
    a.grad_x, a.grad_y = dx.data_ptr(), dy.data_ptr()
    part = buf.new(lib.norm_wait_bytes(C.byref(a)) // 4, dtype=torch.float32)
    assert lib.norm_wait_bwd(C.byref(a), C.c_void_p(part.data_ptr()), stream) == 0
    torch.cuda.synchronize()
    assert status.item() == L.OSSM_ETIMEOUT and buf.intact()
    after = O.residual_norm(x, y, w, post_norm="rms" if post else None)
    assert all(torch.equal(p, q) for p, q in zip(before, after))
    assert O.workspace_status() == 0
