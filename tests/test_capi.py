"""C-ABI library: loads, exports every symbol include/orthossm_b200.h declares,
struct layouts agree with the ctypes binding, argument checks reject bad input
without touching a GPU."""
import ctypes as C
import os
import re

import pytest

from orthossm_b200 import _lib as L

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def declared_symbols():
    src = open(os.path.join(ROOT, "include", "orthossm_b200.h")).read()
    src = re.sub(r"/\*.*?\*/", "", src, flags=re.S)
    return sorted(set(re.findall(r"\b(ossm_[a-z0-9_]+)\s*\(", src)))


def test_header_matches_binding_list():
    assert declared_symbols() == sorted(L.EXPORTED)


def test_library_loads_and_exports_all():
    lib = L.lib()
    for name in declared_symbols():
        assert hasattr(lib, name), name
    assert b"sm_100a" in lib.ossm_version()


def test_struct_layouts():
    lib = L.lib()
    assert lib.ossm_sizeof_fwd_args() == C.sizeof(L.FwdArgs)
    assert lib.ossm_sizeof_lion_args() == C.sizeof(L.LionArgs)


def test_status_strings():
    lib = L.lib()
    for s in range(6):
        assert lib.ossm_status_string(s)


def _args(**kw):
    a = dict(B=1, S=16, H=8, head_dim=64, degree=8, x=4096, x_dtype=L.OSSM_BF16, x_stride_b=16 * 512,
             x_stride_s=512, coeffs=8192, out=16384, out_dtype=L.OSSM_BF16, out_stride_b=16 * 512,
             out_stride_s=512, momentum=0.9)
    a.update(kw)
    return L.FwdArgs(**a)


def test_workspace_size_and_validation():
    lib = L.lib()
    ok = _args()
    n = lib.ossm_fwd_workspace_bytes(C.byref(ok))
    assert n > 256 and n % 256 == 0
    bad = [_args(head_dim=48), _args(head_dim=4), _args(degree=9), _args(degree=0), _args(S=0),
           _args(x=4098), _args(x_stride_s=100), _args(flags=3), _args(flags=L.OSSM_EVAL_LUT),
           _args(out_dtype=7), _args(gate_w=4096)]
    for a in bad:
        assert lib.ossm_fwd_workspace_bytes(C.byref(a)) == 0
        # rejected before any CUDA call
        assert lib.ossm_cheby_ema_fwd(C.byref(a), None, 0, None) == L.OSSM_EINVAL
    assert lib.ossm_cheby_ema_fwd(C.byref(ok), None, 0, None) == L.OSSM_EWORKSPACE


def test_gate_workspace_grows_with_tokens():
    lib = L.lib()
    a = _args(gate_w=4096, gate_b=4096, lam_h=4096)
    b = _args(S=32, x_stride_b=32 * 512, out_stride_b=32 * 512, gate_w=4096, gate_b=4096, lam_h=4096)
    assert lib.ossm_fwd_workspace_bytes(C.byref(b)) > lib.ossm_fwd_workspace_bytes(C.byref(a))


def test_lion_validation():
    lib = L.lib()
    a = L.LionArgs(B=1, S=16, H=8, head_dim=8, degree=4, chunk=0, x=4096, x_dtype=L.OSSM_F32,
                   x_stride_b=16 * 64, x_stride_s=64, coeffs=8192, momentum=8192, out=4096,
                   out_dtype=L.OSSM_F32, out_stride_b=16 * 64, out_stride_s=64)
    assert lib.ossm_cheby_rkv_lion(C.byref(a), None) == L.OSSM_EINVAL
    a.chunk = 8
    a.flags = L.OSSM_EVAL_LUT  # LUT mode without a table
    assert lib.ossm_cheby_rkv_lion(C.byref(a), None) == L.OSSM_EINVAL


def test_ops_refuse_cpu_tensors():
    import torch
    from orthossm_b200 import cheby_ema_forward
    with pytest.raises(RuntimeError, match="CUDA"):
        cheby_ema_forward(torch.zeros(1, 8, 64), torch.zeros(1, 8, 8, 8))


def test_host_workspace_size_and_validation():
    """ossm_fwd_host_workspace_bytes: the device forward's workspace for the
    largest part plus the part plan's staging buffers; no GPU needed."""
    lib = L.lib()
    B, S = 8, 4096
    base = dict(B=B, S=S, x_stride_b=S * 512, out_stride_b=S * 512)
    n8 = lib.ossm_fwd_host_workspace_bytes(C.byref(_args(**base)), 8)
    n16 = lib.ossm_fwd_host_workspace_bytes(C.byref(_args(**base)), 16)
    one_part = S * 512 * 2  # one sequence of bf16 activations
    assert n8 % 256 == 0 and n8 >= 2 * 2 * one_part  # two x and two out buffers of one sequence each
    assert n16 < n8  # 16 parts: half sequences
    assert lib.ossm_fwd_host_workspace_bytes(C.byref(_args(**base)), 1) >= 2 * 2 * B * one_part
    bad = [(_args(**base), 0), (_args(**dict(base, x_stride_b=S * 512 + 512)), 8),
           (_args(**dict(base, out_stride_s=1024)), 8), (_args(**dict(base, tanh_out=4096)), 8),
           (_args(**dict(base, degree=9)), 8)]
    for a, pieces in bad:
        assert lib.ossm_fwd_host_workspace_bytes(C.byref(a), pieces) == 0
    assert lib.ossm_cheby_ema_fwd_host(C.byref(_args(**base)), 8, None, 0, None) == L.OSSM_EWORKSPACE
    assert lib.ossm_cheby_ema_fwd_host(C.byref(_args(**dict(base, tanh_out=4096))), 8, None, 0, None) == L.OSSM_EINVAL


def _attn(**kw):
    a = dict(B=1, H=4, H_kv=2, head_dim=64, total_q=8, total_k=8, max_seqlen_q=8, dtype=L.OSSM_BF16, q=4096, k=4096,
             v=4096, out=4096, q_stride_t=256, q_stride_h=64, k_stride_t=128, k_stride_h=64, v_stride_t=128,
             v_stride_h=64, out_stride_t=256, out_stride_h=64, cu_q=4096, cu_k=4096, scale=1.0)
    a.update(kw)
    return L.AttnArgs(**a)


def test_attention_workspace_has_one_size():
    """A larger one for some arguments would replace the one that captured
    graphs point to."""
    lib = L.lib()
    sizes = {lib.ossm_attn_workspace_bytes(C.byref(_attn(**kw)))
             for kw in (dict(), dict(head_dim=8), dict(head_dim=128, q_stride_h=128, k_stride_h=128, v_stride_h=128,
                                                       out_stride_h=128), dict(H=2, total_q=1, max_seqlen_q=1))}
    assert len(sizes) == 1 and sizes.pop() > L.OSSM_ATTN_WS_ZERO
    assert lib.ossm_attn_workspace_bytes(C.byref(_attn(head_dim=136))) == 0
    src = open(os.path.join(ROOT, "include", "orthossm_b200.h")).read()
    assert int(re.search(r"#define OSSM_ATTN_WS_ZERO (\d+)", src).group(1)) == L.OSSM_ATTN_WS_ZERO
    assert lib.ossm_stream_capture_id(None, None) == L.OSSM_EINVAL


def test_attention_workspace_under_capture(monkeypatch):
    """One workspace a stream outside captures, kept for good; one a graph and
    stream within, zero-filled in the graph."""
    import types

    import torch

    from orthossm_b200 import sdpc_kernel, serving
    now = [0]

    class Lib:
        def ossm_stream_capture_id(self, stream, ref):
            ref._obj.value = now[0]
            return L.OSSM_OK

    monkeypatch.setattr(L, "lib", Lib)
    for d in (sdpc_kernel._WS_ATTN, sdpc_kernel._WS_CAPTURED):
        for key in [k for k in d if torch.device("cpu") in k]:
            del d[key]
    s, t = types.SimpleNamespace(cuda_stream=1), types.SimpleNamespace(cuda_stream=2)
    get = lambda st, c: serving._attn_workspace(torch.device("cpu"), st, 1 << 17, c)  # noqa: E731
    own = get(s, False)
    assert get(s, False) is own and get(t, False) is not own and int(own.sum()) == 0
    now[0] = 5
    first, side = get(s, True), get(t, True)
    assert first is not own and side is not first and get(s, True) is first
    assert int(first[:L.OSSM_ATTN_WS_ZERO].sum()) == 0
    now[0] = 6
    second = get(s, True)
    assert second is not first and second is not own and get(s, True) is second
    assert get(s, False) is own


def test_workspaces_that_graphs_use_are_kept(monkeypatch):
    """The other operators' workspaces grow: one that a captured call was given
    stays alive, and captured calls without one get their graph's own."""
    import types

    import torch

    from orthossm_b200 import sdpc_kernel as K
    on = [False]

    class Lib:
        def ossm_stream_capture_id(self, stream, ref):
            ref._obj.value = 9
            return L.OSSM_OK

    monkeypatch.setattr(L, "lib", Lib)
    monkeypatch.setattr(K, "_is_capturing", lambda: on[0])
    monkeypatch.setattr(K, "_WS", {})
    monkeypatch.setattr(K, "_WS_CAPTURED", {})
    monkeypatch.setattr(K, "_WS_IN_GRAPHS", [])
    s, t = types.SimpleNamespace(cuda_stream=1), types.SimpleNamespace(cuda_stream=2)
    get = lambda st, n: K._workspace(torch.device("cpu"), st, n)  # noqa: E731
    small = get(s, 1 << 17)
    on[0] = True
    assert get(s, 1 << 17) is small and get(s, 1 << 16) is small
    larger = get(s, 1 << 18)  # within the capture
    fresh = get(t, 1 << 16)
    assert larger is not small and get(s, 1 << 18) is larger and get(t, 1 << 16) is fresh
    assert int(larger.sum()) == 0
    on[0] = False
    grown = get(s, 1 << 19)
    assert grown is not small and grown is not larger and get(s, 1 << 17) is grown
    assert len(K._WS_IN_GRAPHS) == 1 and K._WS_IN_GRAPHS[0] is small
    assert get(t, 1 << 16) is not fresh


def test_attention_counters_do_not_overlap():
    """Two counters a CTA and one for the second step, of up to 4 CTAs on each
    of the SMs that are used, within what the caller zero-fills."""
    src = open(os.path.join(ROOT, "orthossm_b200", "csrc", "ossm_attn.cuh")).read()
    sms = int(re.search(r"kMaxSms = (\d+)", src).group(1))
    assert sms >= 148 and 256 + 3 * 4 * sms * 4 <= L.OSSM_ATTN_WS_ZERO
    assert L.lib().ossm_attn_workspace_bytes(C.byref(_attn())) > 256 + 3 * 4 * sms * 4


def test_sampling_limits():
    """Refused before any CUDA call."""
    lib = L.lib()
    f = lambda **kw: lib.ossm_sample_tokens(C.byref(L.SampleArgs(  # noqa: E731
        **{**dict(B=1, V=8, logits=4096, dtype=L.OSSM_F32, logits_stride=8, inv_temperature=1.0, top_p=1.0,
                  out=4096), **kw})), None)
    for bad in (dict(V=1 << 23), dict(V=0), dict(B=(1 << 27) + 1), dict(B=-1), dict(logits=0), dict(logits=4097),
                dict(out=4), dict(dtype=7), dict(top_p=-0.5), dict(min_p=float("nan")), dict(top_k=-1)):
        assert f(**bad) == L.OSSM_EINVAL, bad
    assert f(B=0) == L.OSSM_OK


def test_attention_flags():
    lib = L.lib()
    src = open(os.path.join(ROOT, "include", "orthossm_b200.h")).read()
    assert int(re.search(r"#define OSSM_ATTN_NO_CAPTURE (\d+)u", src).group(1)) == L.OSSM_ATTN_NO_CAPTURE
    assert lib.ossm_attn_workspace_bytes(C.byref(_attn(flags=1))) > 0
    assert lib.ossm_attn_workspace_bytes(C.byref(_attn(flags=2))) == 0
