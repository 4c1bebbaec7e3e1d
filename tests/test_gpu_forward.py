"""GPU parity of the fused forward (ossm_cheby_ema_fwd) against the oracle and
the reference's golden outputs.

Tolerances: fp32 I/O 1e-5 relative (norm-wise);
bf16 I/O with fp32 state 2e-2 relative.  The parallel scan's reassociation
and, for bf16 output, tanh.approx + bf16 rounding are the tolerance sources.
"""
import numpy as np
import pytest
import torch

from oracle import cheby_ref as R
from tests.golden.inputs import det_normal, linear_init, spectral_coeffs
from tests.test_oracle_golden import load, relerr

pytestmark = pytest.mark.gpu
dev = "cuda"
F32_TOL = 1e-5
BF16_TOL = 2e-2


def f32(v):
    """Decays as the kernel receives them (fp32): the EMA amplifies a decay
    error by ~1/(1-lambda), so the oracle must see the same fp32 values."""
    return np.asarray(v, np.float32).astype(np.float64)


def T(a, dtype=torch.float32):
    return torch.from_numpy(np.ascontiguousarray(a)).to(dev, dtype)


def N(t):
    return t.detach().float().cpu().numpy().astype(np.float64)


def run(x, c, **kw):
    import orthossm_b200 as O
    return O.cheby_ema_forward(x, c, **kw)


# ---------------------------------------------------------------- fp32 pins

def test_config1_fp32_per_head_lambda():
    """fp32, B=1, S=2048, D=512, deg 8, per-head lambda."""
    g = load("cfg1")
    x = det_normal((1, 2048, 512), 1)
    c = spectral_coeffs(1, 8, 8, 64, 2)
    out, fin = run(T(x), T(c), lambda_per_head=g["lam"].tolist())
    o = N(out)
    assert relerr(o[:, g["rows"]], g["out_rows"]) < F32_TOL
    assert relerr(N(fin), g["final"]) < F32_TOL
    ref = R.cheby_ema_forward(x, c, lam=f32(g["lam"]))
    assert relerr(o, ref["out"]) < F32_TOL
    assert np.abs(o - ref["out"]).max() < 1e-5


@pytest.mark.parametrize("name", ["fused_f32_deg8", "fused_f32_deg4_init"])
def test_fused_kernel_goldens(name):
    g = load(name)
    B, S, D = (int(v) for v in g["shape"])
    H, K = int(g["H"]), int(g["K"])
    x = det_normal((B, S, D), int(g["seed_x"]))
    c = spectral_coeffs(B, H, K, D // H, int(g["seed_c"]), scale=1.0 if K == 8 else 1.5)
    init = g.get("init")
    out, fin, th = run(T(x), T(c), ema_momentum=float(g["momentum"]),
                       init_state=None if init is None else T(init), return_tanh=True)
    assert relerr(N(out), g["out"]) < F32_TOL
    assert relerr(N(th), g["tanh"]) < F32_TOL
    assert relerr(N(fin), g["final"]) < F32_TOL


def test_lut_mode_golden():
    g = load("fused_lut_deg8")
    x = det_normal((1, 200, 64), 121)
    c = spectral_coeffs(1, 4, 8, 16, 122)
    out, fin = run(T(x), T(c), ema_momentum=0.9, eval_mode="lut")
    assert relerr(N(out), g["out"]) < F32_TOL
    assert relerr(N(fin), g["final"]) < F32_TOL


def test_nan_zero_inputs_golden():
    g = load("fused_nan")
    out, _, th = run(T(g["x"]), T(g["c"]), ema_momentum=0.9, return_tanh=True)
    nan = np.isnan(g["x"])
    assert np.all(N(th)[nan] == 0.0)
    assert np.isfinite(N(out)).all()
    assert relerr(N(out), g["out"]) < F32_TOL


def test_fast_path_semantics_golden():
    g = load("fast_path")
    x = det_normal((2, 100, 64), 181)
    c = spectral_coeffs(2, 8, 4, 8, 182)
    out, _ = run(T(x), T(c), ema_momentum=0.9, fast_path_semantics=True)
    assert relerr(N(out), g["out"]) < F32_TOL


# ---------------------------------------------------------------- bf16 / gate

def _cfg2_like(B, S, D=512, H=8, seed=10):
    x = R.bf16_round(det_normal((B, S, D), seed)).astype(np.float32)
    c = spectral_coeffs(B, H, 8, D // H, seed + 1)
    W, b = linear_init(H, D, seed + 2)
    init = det_normal((B, D), seed + 3, 0.1)
    return x, c, W, b, init


@pytest.mark.parametrize("B,S", [(2, 3000), (1, 16384), (1, 40001)])
def test_bf16_gate_carried_state(B, S):
    """BASELINE configs[1] semantics at reduced size: bf16 I/O, fp32 state,
    per-token dynamic lambda from Linear(512->8), carried state ~N(0, 0.1).
    S = 40001 gives 1251 chunks per chain: three carry blocks of 512 chunks,
    the last one and the last chunk ragged."""
    x, c, W, b, init = _cfg2_like(B, S)
    lam = f32(R.BASELINE_LAMBDA)
    out, fin = run(T(x, torch.bfloat16), T(c), lambda_per_head=lam.tolist(), gate_weight=T(W),
                   gate_bias=T(b), init_state=T(init))
    assert out.dtype == torch.bfloat16
    ref = R.cheby_ema_forward(x, c, lam=lam, gate=dict(W=W, b=b), init=init)
    assert relerr(N(out), ref["out"]) < BF16_TOL
    assert np.abs(N(out) - ref["out"]).max() < 2e-2
    assert relerr(N(fin), ref["final"]) < BF16_TOL


def test_bf16_precise_flag_tightens():
    """fp32 output of the gated path.  The per-token decay is formed in fp32
    on the device (the oracle forms it in fp64 from the same inputs); its
    rounding (~6e-8) is amplified by ~1/(1-lambda) in the EMA, which bounds the
    agreement at a few 1e-5 here, far inside the 2e-2 bf16 bar."""
    x, c, W, b, init = _cfg2_like(1, 2048, seed=30)
    lam = f32(R.BASELINE_LAMBDA)
    ref = R.cheby_ema_forward(x, c, lam=lam, gate=dict(W=W, b=b), init=init)
    kw = dict(lambda_per_head=lam.tolist(), gate_weight=T(W), gate_bias=T(b), init_state=T(init),
              out_dtype=torch.float32)
    out, fin = run(T(x, torch.bfloat16), T(c), **kw)
    assert relerr(N(out), ref["out"]) < 3e-4
    assert relerr(N(fin), ref["final"]) < 3e-4


# ---------------------------------------------------------------- shapes / edges

@pytest.mark.parametrize("hd,H,K,S", [(8, 8, 8, 300), (16, 8, 4, 1025), (32, 4, 6, 777), (128, 2, 8, 300),
                                      (256, 1, 3, 100), (64, 8, 1, 1), (64, 8, 8, 257), (8, 2, 2, 5000)])
def test_shapes_fp32(hd, H, K, S):
    B = 3
    D = H * hd
    x = det_normal((B, S, D), 40 + hd)
    c = spectral_coeffs(B, H, K, hd, 41 + K)
    init = np.clip(det_normal((B, D), 42, 0.3), -0.99, 0.99)
    lam = f32(np.linspace(0.9, 0.999, H))
    out, fin = run(T(x), T(c), lambda_per_head=lam.tolist(), init_state=T(init))
    ref = R.cheby_ema_forward(x, c, lam=lam, init=init)
    assert relerr(N(out), ref["out"]) < F32_TOL
    assert relerr(N(fin), ref["final"]) < F32_TOL


def test_init_outside_unit_interval_first_step_clamp():
    """A carried state outside [-1, 1] is clamped by the first step, after
    which the scan is linear (per-step-clamp semantics)."""
    x = det_normal((1, 600, 64), 50)
    c = spectral_coeffs(1, 8, 8, 8, 51)
    init = np.where(np.arange(64) % 2 == 0, 3.0, -2.5)[None].astype(np.float32)
    out, fin = run(T(x), T(c), ema_momentum=0.97, init_state=T(init))
    ref = R.cheby_ema_forward(x, c, momentum=f32(0.97), init=init)
    assert np.abs(N(out)).max() <= 1.0
    assert relerr(N(out), ref["out"]) < F32_TOL


def test_strided_input_and_output():
    base = T(det_normal((2, 700, 1024), 60))
    x = base[:, :, 256:768]  # row stride 1024, channel stride 1
    c = T(spectral_coeffs(2, 8, 8, 64, 61))
    out_full = torch.zeros(2, 700, 2048, device=dev)
    out = out_full[:, :, 512:1024]
    run(x, c, ema_momentum=0.95, out=out)
    ref = R.cheby_ema_forward(N(x), N(c), momentum=f32(0.95))
    assert relerr(N(out), ref["out"]) < F32_TOL
    assert float(out_full[:, :, :512].abs().max()) == 0.0


def test_long_chain_lookback():
    """Many chunks per (b, h) chain: exercises the decoupled look-back."""
    S = 65536
    x = R.bf16_round(det_normal((1, S, 512), 70))
    c = spectral_coeffs(1, 8, 8, 64, 71)
    lam = f32(R.BASELINE_LAMBDA)
    out, fin = run(T(x), T(c), lambda_per_head=lam.tolist(), out_dtype=torch.float32)
    ref = R.cheby_ema_forward(x, c, lam=lam)
    assert relerr(N(out), ref["out"]) < F32_TOL
    assert relerr(N(fin), ref["final"]) < F32_TOL
    import orthossm_b200 as O
    assert O.workspace_status() == 0


@pytest.mark.parametrize("generic", [True, False])
def test_deterministic_and_workspace_reuse(generic):
    """Both the generic kernel and the bf16 fast path (here the cluster
    kernel: four sequences) fold their carries in a fixed order, so a repeat
    call is bitwise the first, also after another shape reused the
    workspace."""
    x, c, W, b, init = _cfg2_like(4, 8192, seed=80)
    kw = dict(lambda_per_head=R.BASELINE_LAMBDA, gate_weight=T(W), gate_bias=T(b), init_state=T(init),
              force_generic=generic)
    xb = T(x, torch.bfloat16)
    o1, f1 = run(xb, T(c), **kw)
    # a different shape in between reuses (and grows) the same workspace
    run(T(det_normal((1, 333, 64), 81)), T(spectral_coeffs(1, 8, 8, 8, 82)))
    o2, f2 = run(xb, T(c), **kw)
    assert torch.equal(o1, o2) and torch.equal(f1, f2)


def test_streaming_chunks_equal_single_call():
    """Streaming in chunks with the carried state (configs[2] pattern)
    reproduces the single-call scan."""
    S, chunk = 20000, 4096
    x = R.bf16_round(det_normal((1, S, 512), 90))
    c = T(spectral_coeffs(1, 8, 8, 64, 91))
    lam = R.BASELINE_LAMBDA
    xf = T(x)
    full, fin = run(xf, c, lambda_per_head=lam)
    state = None
    parts = []
    for t0 in range(0, S, chunk):
        o, state = run(xf[:, t0:t0 + chunk], c, lambda_per_head=lam, init_state=state)
        parts.append(o)
    assert relerr(N(torch.cat(parts, 1)), N(full)) < 1e-6
    assert relerr(N(state), N(fin)) < 1e-6


def test_final_state_is_last_output_fp32():
    x = T(det_normal((2, 1000, 256), 95))
    c = T(spectral_coeffs(2, 4, 8, 64, 96))
    out, fin = run(x, c, ema_momentum=0.99)
    assert torch.equal(out[:, -1, :], fin)


@pytest.mark.parametrize("path", ["default", "generic", "fp32_out"])
def test_nan_inf_and_huge_inputs(path):
    """The reference's fused semantics at non-finite and huge inputs
    (sdpc_kernel.py:1078-1085, :1160-1164): NaN x contributes u = 0 (also at
    token 0 of the sequence, where the carried-in state is folded in with a
    clamp), +-inf and |x| near the bf16 maximum give xn = +-1."""
    from orthossm_b200 import _lib as L
    B, S, D, H = 4, 200, 512, 8
    x = R.bf16_round(det_normal((B, S, D), 91)).astype(np.float32)
    x[0, 5, 3] = np.nan
    x[1, 17, 100] = np.inf
    x[2, 150, 511] = -np.inf
    x[3, 0, :7] = np.nan
    x[3, 199, 64] = 3.0e38
    x[2, 0, 8] = -np.inf
    c = spectral_coeffs(B, H, 8, 64, 92).astype(np.float32)
    init = det_normal((B, D), 93, 0.1).astype(np.float32)
    lam = np.asarray(R.BASELINE_LAMBDA, np.float32)
    kw = dict(lambda_per_head=lam.tolist(), init_state=T(init))
    if path == "generic":
        kw["force_generic"] = True
    if path == "fp32_out":
        kw["out_dtype"] = torch.float32
    from orthossm_b200.sdpc_kernel import _cheby_ema_forward
    out, fin = _cheby_ema_forward(T(x, torch.bfloat16), T(c), **kw)
    ref = R.cheby_ema_forward(x, c, lam=f32(lam), init=init)
    o = N(out)
    assert np.isfinite(o).all() and np.isfinite(N(fin)).all()
    assert relerr(o, ref["out"]) < BF16_TOL
    assert relerr(N(fin), ref["final"]) < BF16_TOL


@pytest.mark.parametrize("mode", ["gate", "lamtok", "f32out"])
def test_two_stream_batch_split_is_bitwise_the_per_sequence_result(mode):
    """B = 4 x S = 16384 runs split over several streams: bf16 outputs as
    slabs of one sequence with u parked in L2 (fp16), fp32 outputs as two
    halves.  Every row must be bitwise what a launch of that sequence alone
    gives, carried state included.  The one-stream launch (OSSM_F_ONE_STREAM)
    evaluates u twice in fp32 instead of parking it: bitwise equal for fp32
    outputs, within one bf16 step (2^-7 relative, 5e-4 absolute near zero)
    and 1e-5 on the final state for bf16."""
    B, S = 4, 16384
    x, c, W, b, init = _cfg2_like(B, S, seed=60)
    xb, cb, ib = T(x, torch.bfloat16), T(c), T(init)
    kw = dict(lambda_per_head=R.BASELINE_LAMBDA.tolist() if hasattr(R.BASELINE_LAMBDA, "tolist")
              else list(R.BASELINE_LAMBDA))
    lt = None
    if mode == "gate":
        kw.update(gate_weight=T(W), gate_bias=T(b))
    if mode == "lamtok":
        lt = (0.99 + 0.01 * torch.rand(B, S, 8, generator=torch.Generator().manual_seed(3))).to(dev)
    odt = torch.float32 if mode == "f32out" else torch.bfloat16
    from orthossm_b200 import _lib as L
    from orthossm_b200.sdpc_kernel import _cheby_ema_forward
    tp = 0  # the default three-pass kernels, which split the batch
    out, fin = _cheby_ema_forward(xb, cb, init_state=ib, out_dtype=odt, lam_tok=lt, extra_flags=tp, **kw)
    # the same launch kept on the caller's stream (OSSM_F_ONE_STREAM)
    o1, f1 = _cheby_ema_forward(xb, cb, init_state=ib, out_dtype=odt, lam_tok=lt,
                                extra_flags=tp | L.OSSM_F_ONE_STREAM, **kw)
    if odt == torch.float32:
        assert torch.equal(out, o1) and torch.equal(fin, f1), mode
    else:
        d = (out.float() - o1.float()).abs()
        assert (d <= 2.0 ** -7 * o1.float().abs() + 5e-4).all(), mode
        assert (fin - f1).abs().max().item() < 1e-5, mode
    for i in range(B):
        oi, fi = _cheby_ema_forward(xb[i:i + 1].contiguous(), cb[i:i + 1].contiguous(),
                                    init_state=ib[i:i + 1].contiguous(), out_dtype=odt,
                                    lam_tok=None if lt is None else lt[i:i + 1].contiguous(), extra_flags=tp, **kw)
        assert torch.equal(out[i:i + 1], oi), (mode, i)
        assert torch.equal(fin[i:i + 1], fi), (mode, i)
    import orthossm_b200 as O
    assert O.workspace_status() == 0


@pytest.mark.parametrize("gate", [True, False])
def test_long_single_sequence_runs_as_two_ranges(gate):
    """B = 1 x S = 131849 (4121 chunks) runs as two token ranges on two
    streams, the second taking the first's end state as its carry-in.  The
    one-stream launch (OSSM_F_ONE_STREAM; oracle-checked at smaller sizes)
    is the reference: outputs within bf16 shard tolerance, the final state to
    fp32 rounding of the carries, and the first four 512-chunk blocks (whose
    carries fold identically in both) bitwise."""
    import orthossm_b200 as O
    from orthossm_b200 import _lib as L
    from orthossm_b200.sdpc_kernel import _cheby_ema_forward
    S = 4096 * 32 + 777
    g = torch.Generator().manual_seed(81)
    x = torch.randn(1, S, 512, generator=g).to(torch.bfloat16).to(dev)
    c = (torch.randn(1, 8, 8, 64, generator=g) / torch.arange(1, 9).view(1, 1, 8, 1)).to(dev)
    init = (0.1 * torch.randn(1, 512, generator=g)).to(dev)
    kw = dict(lambda_per_head=list(R.BASELINE_LAMBDA), init_state=init)
    if gate:
        kw.update(gate_weight=((torch.rand(8, 512, generator=g) * 2 - 1) / 512 ** 0.5).to(dev),
                  gate_bias=((torch.rand(8, generator=g) * 2 - 1) / 512 ** 0.5).to(dev))
    out, fin = run(x, c, **kw)
    o1, f1 = _cheby_ema_forward(x, c, extra_flags=L.OSSM_F_ONE_STREAM, **kw)
    assert (out.float() - o1.float()).abs().max().item() <= 2 ** -7
    assert relerr(N(fin), N(f1)) < 1e-5
    head = 4 * 512 * 32
    assert torch.equal(out[:, :head], o1[:, :head])
    assert O.workspace_status() == 0


def test_graph_outlives_a_larger_workspace():
    """A captured forward, replayed after a longer one on the same stream has
    taken a larger workspace and the freed memory was overwritten; and one
    captured on a stream that has seen no call."""
    import orthossm_b200 as O
    mk = lambda S: torch.randn(2, S, 512, device="cuda").to(torch.bfloat16)  # noqa: E731
    x, far = mk(4096), mk(65536)
    c = O.init_chebyshev_coefficients(2, 8, 8, 64, "cuda")
    gate = dict(lambda_per_head=T(R.BASELINE_LAMBDA), gate_weight=torch.randn(8, 512, device="cuda") * 0.02,
                gate_bias=torch.zeros(8, device="cuda"))
    want, fin = O.cheby_ema_forward(x, c, **gate)
    for before in (True, False):
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        if before:
            with torch.cuda.stream(side):
                O.cheby_ema_forward(x, c, **gate)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out, f = O.cheby_ema_forward(x, c, **gate)
        with torch.cuda.stream(side):
            O.cheby_ema_forward(far, c, **gate)
            waste = [torch.full((1 << 26,), 0x5a5a5a5a, dtype=torch.int32, device="cuda") for _ in range(4)]
        torch.cuda.synchronize()
        del waste
        for _ in range(3):
            out.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want) and torch.equal(f, fin)
    assert O.workspace_status() == 0
