"""fp8 layer kernels against 64-bit references: quantisation, norm, block-scaled products."""
import pytest
import torch

from nanovllm_self_b200.ops import torch_ref as R

pytestmark = pytest.mark.gpu

DEV = "cuda"
U = 2.0 ** -24  # half a step of fp32, relative


@pytest.fixture(scope="module")
def ops():
    from nanovllm_self_b200.ops import get_ops
    return get_ops(DEV)


@pytest.fixture(autouse=True)
def _no_device_error():
    yield
    from nanovllm_self_b200.ops._ext import load
    torch.cuda.synchronize()
    assert load().fp8_error(True) == 0


def _acts(t, k, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    c = torch.exp(torch.randn(k, device=DEV, generator=g))
    return (torch.randn(t, k, device=DEV, generator=g) * c).to(torch.bfloat16)


def _weight(n, k, seed=1):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return R.quant_fp8_weight(0.02 * torch.randn(n, k, device=DEV, generator=g))


def _bits(q):
    return q.view(torch.uint8)


def _same_pair(got, want):
    assert torch.equal(_bits(got[0]), _bits(want[0]))
    assert torch.equal(got[1], want[1])


def _check_quantised(q, s, y, rel):
    """(q, s) stands for the 64-bit values y up to `rel` of fp32 arithmetic and half a step of e4m3."""
    t, k = y.shape
    kb = -(-k // 128)
    p = y.new_zeros(t, kb * 128)
    p[:, :k] = y.abs()
    want = p.view(t, kb, 128).amax(-1).clamp(min=R.FP8_AMAX_MIN) / 448.0
    assert ((s.double() - want).abs() <= rel * want).all()
    sc = s.double().repeat_interleave(128, 1)[:, :k]
    err = (q.double() * sc - y).abs()
    # half a step: 2^-4 of a normal value, 2^-10 of the scale below e4m3's smallest normal
    assert (err <= y.abs() * (2.0 ** -4 + 2 * rel) + sc * 2.0 ** -10 * (1 + rel)).all()


# --------------------------------------------------------------------------- quantisation
@pytest.mark.parametrize("t,k", [(1, 16), (1, 4096), (3, 128), (17, 144), (16, 512), (33, 1712), (257, 4096),
                                 (1000, 640), (4097, 208)])
def test_quant_matches_definition(ops, t, k):
    x = _acts(t, k)
    got = ops.quant_fp8(x)
    assert got[0].shape == (t, k) and got[1].shape == (t, -(-k // 128))
    _same_pair(got, R.quant_fp8(x))                 # the same fp32 operations: bit for bit
    _check_quantised(*got, x.double(), 4 * U)


def test_quant_zeros_extremes_and_nonfinite(ops):
    x = torch.zeros(6, 256, dtype=torch.bfloat16, device=DEV)
    x[1] = torch.finfo(torch.bfloat16).max
    x[1, ::2] *= -1
    x[2] = 1e-38                                    # below the floor of the group maximum
    x[3, 5] = float("inf")
    x[4, 130] = float("nan")
    x[5, 0] = -3.0
    q, s = ops.quant_fp8(x)
    _same_pair((q[[0, 1, 2, 5]], s[[0, 1, 2, 5]]), tuple(v[[0, 1, 2, 5]] for v in R.quant_fp8(x)))
    d = R.dequant_fp8(q, s)
    assert (d[0] == 0).all() and torch.isfinite(d[[0, 1, 2, 5]]).all()
    assert torch.isnan(d[3, :128]).all() and (d[3, 128:] == 0).all()   # its own group only
    assert torch.isnan(d[4, 128:]).all() and (d[4, :128] == 0).all()


def test_quant_row_stride(ops):
    big = _acts(40, 512)
    x = big[::2, 128:384]
    _same_pair(ops.quant_fp8(x), R.quant_fp8(x))
    assert ops.quant_fp8(x[:0])[0].shape == (0, 256)


# --------------------------------------------------------------------------- norm
@pytest.mark.parametrize("residual", [True, False])
@pytest.mark.parametrize("t,k", [(1, 16), (1, 4096), (5, 144), (256, 4096), (63, 5120), (7, 8192), (3, 16384),
                                 (300, 2064), (2, 10000)])
def test_norm(ops, t, k, residual):
    eps = 1e-6
    x, w = _acts(t, k), (1 + 0.1 * torch.randn(k, device=DEV)).to(torch.bfloat16)
    res = _acts(t, k, 7) if residual else None
    want_r = x if res is None else (x.float() + res.float()).to(torch.bfloat16)
    (q, s), r = ops.add_rmsnorm_fp8(x, None if res is None else res, w, eps)
    assert r.data_ptr() == (x if res is None else res).data_ptr()
    assert torch.equal(r, want_r)
    d = want_r.double()
    y = d / torch.sqrt(d.square().mean(1, keepdim=True) + eps) * w.double()
    # sum of squares: 64 terms in a row per thread, then 5 + 8 additions; half of that relative error
    # passes the root; rsqrt (2 units), two products and a division
    _check_quantised(q, s, y, ((64 + 13 + 2) / 2 + 8) * U)


@pytest.mark.parametrize("eps", [0.0, 1e-6])
def test_norm_group_of_zero_weights_and_tiny_rows(ops, eps):
    """A group below the floor beside ordinary ones, its factor past fp32's range without eps."""
    x = (_acts(5, 512).float() * 1e-9).to(torch.bfloat16)
    w = torch.ones(512, device=DEV, dtype=torch.bfloat16)
    w[128:256] = 0
    (q, s), _ = ops.add_rmsnorm_fp8(x, None, w, eps)
    d = x.double()
    _check_quantised(q, s, d / torch.sqrt(d.square().mean(1, keepdim=True) + eps) * w.double(), ((64 + 13 + 2) / 2 + 8) * U)
    assert (q[:, 128:256].float() == 0).all()


def _norm_rel(k):
    """Error of the row's factor and what follows it, relative: 8 squares per thread and step of 1024
    channels are added in a row, then 5 + 4 sums; with a square's own rounding, the mean's division and eps
    8 c + 12, half of which passes the root.  rsqrt is within 2 ulp (4 halves of one); up to two products by
    the factor and w, the division by 448 or of it, and the product with its result."""
    return (4 * -(-k // 1024) + 6 + 4 + 4) * U


def _norm_exact(r, w, eps):
    d = r.double()
    return d / torch.sqrt(d.square().mean(1, keepdim=True) + eps) * w.double()


# every number of vectors per thread that has a kernel of its own, with groups that end inside a step
NORM_K = [256, 2048, 2064, 4096, 5120, 6144, 8192, 10000, 16384]


@pytest.mark.parametrize("residual", [True, False])
@pytest.mark.parametrize("eps", [0.0, 1e-12, 1e-10])
@pytest.mark.parametrize("k", NORM_K)
def test_norm_groups_of_tiny_values(ops, k, eps, residual):
    """Groups between 1e-38 and 1e-18 in rows that a small eps scales up by as much as 1e18: 448 over a
    group's largest |r w| alone would leave fp32's range."""
    g = torch.Generator(device=DEV).manual_seed(k)
    t, kb = 5, -(-k // 128)
    mag = 10.0 ** (-38 + 20 * torch.rand(t, kb, device=DEV, generator=g, dtype=torch.float64))
    mag[:, 0] = 1e-18
    mag[1] = 1e-37                                  # eps alone makes this row's factor, where there is one
    mag[1, 0] = 1e-37 if eps else 1e-18
    v = torch.randn(t, k, device=DEV, generator=g, dtype=torch.float64) * mag.repeat_interleave(128, 1)[:, :k]
    v[0, 128:132] = torch.tensor([1e-37, 5e-38, 0.0, 2e-38], device=DEV, dtype=torch.float64)
    v[0, 132:256] = 0
    x = v.to(torch.bfloat16)
    w = (1 + 0.1 * torch.randn(k, device=DEV, generator=g)).to(torch.bfloat16)
    res = torch.zeros_like(x) if residual else None
    (q, s), _ = ops.add_rmsnorm_fp8(x, res, w, eps)
    _check_quantised(q, s, _norm_exact(x, w, eps), _norm_rel(k))


@pytest.mark.parametrize("k", NORM_K)
def test_norm_weights_whose_product_with_the_row_overflows(ops, k):
    """r w leaves fp32's range where the norm itself does not."""
    x = (_acts(3, k).float() * 1e10).to(torch.bfloat16)
    w = (1 + 0.1 * torch.randn(k, device=DEV, generator=torch.Generator(device=DEV).manual_seed(2))).to(torch.bfloat16)
    w[128:256] *= 1e30
    (q, s), _ = ops.add_rmsnorm_fp8(x, None, w, 1e-6)
    _check_quantised(q, s, _norm_exact(x, w, 1e-6), _norm_rel(k))


def test_norm_infinity_stays_in_its_group(ops):
    x = _acts(2, 512)
    x[0, 130] = float("inf")
    w = torch.ones(512, device=DEV, dtype=torch.bfloat16)
    d = R.dequant_fp8(*ops.add_rmsnorm_fp8(x, None, w, 1e-6)[0])
    # finite values over an infinite root are zero; the group of the infinity itself is not a number
    assert torch.isnan(d[0, 128:256]).all() and (d[0, :128] == 0).all() and (d[0, 256:] == 0).all()
    assert torch.isfinite(d[1]).all()


@pytest.mark.parametrize("k", NORM_K)
def test_norm_within_its_own_error_bound(ops, k):
    x, res = _acts(9, k), _acts(9, k, 7)
    w = (1 + 0.1 * torch.randn(k, device=DEV, generator=torch.Generator(device=DEV).manual_seed(3))).to(torch.bfloat16)
    (q, s), r = ops.add_rmsnorm_fp8(x, res, w, 1e-6)
    _check_quantised(q, s, _norm_exact(r, w, 1e-6), _norm_rel(k))


@pytest.mark.parametrize("t,k", [(64, 4096), (33, 1040)])
def test_norm_values_are_those_of_r_times_w(ops, t, k):
    """r * w is exact in fp32 and the root's factor cancels against the group's maximum, so the 8-bit
    values are those of r * w bit for bit."""
    x, res, w = _acts(t, k), _acts(t, k, 7), (1 + 0.2 * torch.randn(k, device=DEV)).to(torch.bfloat16)
    (q, _), r = ops.add_rmsnorm_fp8(x, res, w, 1e-6)
    assert torch.equal(_bits(q), _bits(R.quant_fp8(r.float() * w.float())[0]))


def test_norm_zero_row_and_nan_row(ops):
    x = _acts(3, 256)
    x[1] = 0
    x[2, 3] = float("nan")
    w = torch.ones(256, device=DEV, dtype=torch.bfloat16)
    (q, s), _ = ops.add_rmsnorm_fp8(x, None, w, 1e-6)
    d = R.dequant_fp8(q, s)
    assert torch.isfinite(d[0]).all() and (d[1] == 0).all() and torch.isnan(d[2]).all()


# --------------------------------------------------------------------------- products
def _bound(x, w):
    """Sum of the magnitudes of every product: what the accumulation's rounding errors scale with."""
    return torch.einsum("tk,nk->tn", R.dequant_fp8(*x, torch.float64).abs(), R.dequant_fp8_weight(*w, torch.float64).abs())


def _exact(x, w):
    return torch.einsum("tk,nk->tn", R.dequant_fp8(*x, torch.float64), R.dequant_fp8_weight(*w, torch.float64))


def _acc(k):
    """Relative error of the sums: 128 products per block, one scaled addition per block, the two
    scales' product."""
    return (128 + 2 * (-(-k // 128)) + 4) * U


SHAPES = [(1, 128, 128), (1, 1, 16), (2, 7, 16), (3, 130, 144), (16, 256, 256), (17, 384, 1712), (33, 250, 640),
          (64, 4096, 512), (65, 512, 4096), (127, 257, 272), (128, 256, 128), (129, 1000, 2064), (256, 640, 4096),
          (300, 129, 528), (513, 2744, 1712), (1, 6144, 4096), (40, 4096, 12288), (1000, 520, 7168)]


@pytest.mark.parametrize("t,n,k", SHAPES)
def test_linear(ops, t, n, k):
    x, w = ops.quant_fp8(_acts(t, k)), _weight(n, k)
    y = ops.linear_fp8(x, w)
    assert y.shape == (t, n) and y.dtype == torch.bfloat16
    want = _exact(x, w)
    assert ((y.double() - want).abs() <= want.abs() * 2.0 ** -8 + 1.01 * _acc(k) * _bound(x, w)).all()


SILU = [(1, 16, 16), (1, 128, 128), (2, 144, 272), (17, 384, 512), (64, 1024, 4096), (100, 2064, 640), (128, 128, 256),
        (129, 272, 1712), (256, 1536, 4096), (700, 400, 528), (1, 12288, 4096)]


@pytest.mark.parametrize("t,i,k", SILU)
def test_linear_silu(ops, t, i, k):
    x = ops.quant_fp8(_acts(t, k))
    g = torch.Generator(device=DEV).manual_seed(3)
    # gates of order one, so that silu's curved part is met
    gu = [torch.randn(i, k, device=DEV, generator=g) / k ** 0.5 for _ in range(2)]
    w = R.quant_fp8_weight(R.group_gate_up(*gu))
    q, s = ops.linear_silu_fp8(x, w, i)
    assert q.shape == (t, i) and s.shape == (t, -(-i // 128))
    y, b = _exact(x, w).view(t, -1, 2, 128), _bound(x, w).view(t, -1, 2, 128)
    gate, up, gb, ub = (v.reshape(t, -1)[:, :i] for v in (y[:, :, 0], y[:, :, 1], b[:, :, 0], b[:, :, 1]))
    h = gate * torch.sigmoid(gate) * up
    # |d silu| <= 1.1 |d gate|, silu <= |gate|; the exponential's argument is off by |gate| U, it by 4 U,
    # the sum by U, the reciprocal by 2 U, two products by U each
    err = 1.01 * _acc(k) * (1.1 * gb * up.abs() + gate.abs() * ub) + (gate.abs() + 9) * U * h.abs()
    kb = -(-i // 128)
    p = h.new_zeros(2, t, kb * 128)
    p[0, :, :i], p[1, :, :i] = h.abs(), err
    want = p[0].view(t, kb, 128).amax(-1).clamp(min=R.FP8_AMAX_MIN)
    worst = p[1].view(t, kb, 128).amax(-1) + 4 * U * want
    assert ((s.double() * 448 - want).abs() <= worst).all()
    sc = s.double().repeat_interleave(128, 1)[:, :i]
    wide = (worst / want).repeat_interleave(128, 1)[:, :i]
    assert ((q.double() * sc - h).abs() <= h.abs() * (2.0 ** -4 + 2 * wide) + 1.1 * err + sc * 2.0 ** -10 * (1 + wide)).all()


def _plans(t, act):
    for np_ in (16, 32) if act else (16, 32, 64):
        if np_ >= t:
            for splits in (1, 2, 3, 5, 8):
                yield [np_, splits]
    yield [-2, 1]
    for splits in (1, 2, 4):
        yield [-1, splits]
        if not act:
            yield [-3, splits]


@pytest.mark.parametrize("t,n,k", [(1, 384, 272), (13, 100, 1712), (32, 640, 1040), (50, 250, 512), (128, 900, 2064), (300, 260, 1312)])
def test_every_kernel_variant(ops, t, n, k):
    """The variants differ in the order of fp32 additions alone."""
    C = ops.C
    x, w = ops.quant_fp8(_acts(t, k)), _weight(n, k)
    want = _exact(x, w)
    tol = want.abs() * 2.0 ** -8 + 1.01 * (_acc(k) + 8 * U) * _bound(x, w)
    for plan in _plans(t, False):
        y = C.linear_fp8(*x, *w, None, plan)
        assert ((y.double() - want).abs() <= tol).all(), plan
    i = (n + 15) // 16 * 16
    g = torch.Generator(device=DEV).manual_seed(3)
    gu = [torch.randn(i, k, device=DEV, generator=g) / k ** 0.5 for _ in range(2)]
    w = R.quant_fp8_weight(R.group_gate_up(*gu))
    q0, s0 = C.linear_silu_fp8(*x, *w, i, [-1, 1])
    d0 = R.dequant_fp8(q0, s0, torch.float64)
    for plan in _plans(t, True):
        q, s = C.linear_silu_fp8(*x, *w, i, plan)
        # scales agree up to the sums' rounding, values up to a step of e4m3
        assert ((s - s0).abs() <= 1e-3 * s0).all(), plan
        step = d0.abs() * 2.0 ** -3 + s0.double().repeat_interleave(128, 1)[:, :i] * 2.0 ** -9
        assert ((R.dequant_fp8(q, s, torch.float64) - d0).abs() <= 1.01 * step + 1e-3 * d0.abs()).all(), plan
        assert (_bits(q) == _bits(q0)).float().mean() > 0.99, plan


def test_plans_refused(ops):
    x, w = ops.quant_fp8(_acts(20, 256)), _weight(256, 256)
    for plan in ([16, 1], [32, 9], [128, 1], [24, 1], [32, 0], [32], [-1, 3], [-1, 8], [-2, 2], [-1, 0], [0, 1], [-4, 1]):
        with pytest.raises(RuntimeError):
            ops.C.linear_fp8(*x, *w, None, plan)
    with pytest.raises(RuntimeError):
        ops.C.linear_silu_fp8(*x, *w, 128, [64, 1])
    with pytest.raises(RuntimeError):
        ops.C.linear_silu_fp8(*x, *w, 128, [-3, 1])


def test_plans_are_those_of_a_process_without_a_gpu(ops):
    """Equal sizes take equal plans, and so give equal bits, in every process."""
    import json
    import os
    import random
    import subprocess
    import sys
    rng = random.Random(0)
    sizes = [(int(2 ** rng.uniform(0, 14)), 16 * int(2 ** rng.uniform(0, 11)), 16 * int(2 ** rng.uniform(0, 10)), rng.random() < 0.3)
             for _ in range(400)] + [(1, 128 * n, 4096, 0) for n in range(1, 300)] + [(256, 128 * n, 8192, 0) for n in range(1, 100)]
    sizes = [[t, -(-n // 256) * 256 if act else n, k, int(act)] for t, n, k, act in sizes]
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    code = ("import json, sys; from nanovllm_self_b200.ops._ext import load; C = load(); "
            f"print(json.dumps([C.fp8_plan(*s, {sms}) for s in json.load(sys.stdin)]))")
    done = subprocess.run([sys.executable, "-c", code], input=json.dumps(sizes), capture_output=True, text=True, timeout=120,
                          env={**os.environ, "CUDA_VISIBLE_DEVICES": ""})
    assert done.returncode == 0, done.stderr[-2000:]
    assert json.loads(done.stdout) == [ops.C.fp8_plan(*s, sms) for s in sizes]


@pytest.mark.parametrize("t", [1, 20, 200])
def test_linear_nan_and_zero_rows_stay_their_own(ops, t):
    k, n = 512, 384
    a = _acts(t + 2, k)
    a[0, 7] = float("nan")
    a[1] = 0
    x, w = ops.quant_fp8(a), _weight(n, k)
    y = ops.linear_fp8(x, w)
    assert torch.isnan(y[0]).all() and (y[1] == 0).all() and torch.isfinite(y[2:]).all()


def test_linear_strides_and_out(ops):
    t, n, k = 70, 272, 512
    a = _acts(t, k)
    q, s = ops.quant_fp8(a)
    wide = torch.zeros(t, 2 * k, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn)
    wide[:, k:].copy_(q)
    w = _weight(n, k)
    want = ops.linear_fp8((q, s), w)
    assert torch.equal(ops.linear_fp8((wide[:, k:], s), w), want)
    for pad, off in ((16, 0), (3, 1), (9, 0)):      # rows that allow 16-byte stores, and rows that do not
        buf = torch.full((t + 1, n + pad), 5.0, dtype=torch.bfloat16, device=DEV)
        out = buf[:t, off:off + n]
        assert ops.linear_fp8((q, s), w, out=out) is not None
        assert torch.equal(out, want)
        assert (buf[t] == 5).all() and (buf[:, :off] == 5).all() and (buf[:, off + n:] == 5).all()


def test_empty_and_single(ops):
    w = _weight(256, 256)
    x = ops.quant_fp8(_acts(5, 256)[:0])
    assert ops.linear_fp8(x, w).shape == (0, 256)
    assert ops.linear_silu_fp8(x, w, 128)[0].shape == (0, 128)


# --------------------------------------------------------------------------- streams and graphs
def _layer(ops, x, res, w, norm):
    """The fp8 part of a decoder layer in its order: norm, product, 8-bit form, product, norm, MLP."""
    h, r = ops.add_rmsnorm_fp8(x, res, norm, 1e-6)
    o = ops.quant_fp8(ops.linear_fp8(h, w["qkv"]))
    y = ops.linear_fp8(o, w["o"])
    h, r = ops.add_rmsnorm_fp8(y, r, norm, 1e-6)
    return ops.linear_fp8(ops.linear_silu_fp8(h, w["gate_up"], 400), w["down"]), r


def _layer_weights(k=512):
    gu = [torch.randn(400, k, device=DEV, generator=torch.Generator(device=DEV).manual_seed(s)) / k ** 0.5
          for s in (5, 6)]
    return {"qkv": _weight(640, k, 1), "o": _weight(k, 640, 2), "gate_up": R.quant_fp8_weight(R.group_gate_up(*gu)),
            "down": _weight(k, 400, 3)}


@pytest.mark.parametrize("t", [1, 37, 300])
def test_layer_matches_plain_layer(ops, t):
    """The operators together, against the plain forms of the same steps run in fp32."""
    from nanovllm_self_b200.ops import TorchOps
    w, norm = _layer_weights(), (1 + 0.1 * torch.randn(512, device=DEV)).to(torch.bfloat16)
    x, res = _acts(t, 512), _acts(t, 512, 9)
    want, want_r = _layer(TorchOps(), x, res.clone(), w, norm)
    got, got_r = _layer(ops, x, res.clone(), w, norm)
    # each step differs by fp32 rounding alone; where that moves a value across the border of an
    # e4m3 step, one operand of the next product moves by up to 2^-3: rare, and averaged over its sum
    for a, b in ((got, want), (got_r, want_r)):
        assert ((a.double() - b.double()).norm() <= 0.01 * b.double().norm())


def test_side_stream_and_concurrent_graphs(ops):
    """No state is shared between calls: two captured layers replayed on two streams at once give
    what the same calls give one after the other."""
    w, norm = _layer_weights(), torch.ones(512, device=DEV, dtype=torch.bfloat16)
    ins = [(_acts(t, 512, t), _acts(t, 512, t + 1)) for t in (3, 200)]
    want = [_layer(ops, x, r.clone(), w, norm)[0] for x, r in ins]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _layer(ops, ins[0][0], ins[0][1].clone(), w, norm)[0]
    torch.cuda.synchronize()
    assert torch.equal(got, want[0])
    graphs = []
    for x, r in ins:
        st = {"r0": r, "r": r.clone(), "x": x}
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            st["r"].copy_(st["r0"])
            st["y"] = _layer(ops, st["x"], st["r"], w, norm)[0]
        graphs.append((g, st))
    streams = [torch.cuda.Stream() for _ in graphs]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(20):
        for (g, _), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for (_, st), y in zip(graphs, want):
        assert torch.equal(st["y"], y)


def test_weights_written_just_before_the_call(ops):
    """The kernels start before the previous kernel ends; what it writes is still seen."""
    x = ops.quant_fp8(_acts(9, 1024))
    pool = [_weight(512, 1024, s) for s in range(6)]
    want = [ops.linear_fp8(x, w) for w in pool]
    q, s = torch.empty_like(pool[0][0]), torch.empty_like(pool[0][1])
    for i in list(range(6)) * 5:
        s.copy_(pool[i][1])
        q.view(torch.uint8).copy_(pool[i][0].view(torch.uint8))
        assert torch.equal(ops.linear_fp8(x, (q, s)), want[i])


@pytest.mark.parametrize("t", [9, 200, 600])
def test_weights_of_a_kernel_that_lets_the_next_one_start_early(ops, t):
    """quant_fp8 signals its dependents before it writes: the product that takes its 8-bit values as weights, and
    starts beside it, sees all of them (one, several and paired CTAs per tile)."""
    n, k = 4096, 2048
    x = ops.quant_fp8(_acts(t, k))
    srcs = [_acts(n, k, s) for s in (11, 12, 13)]
    ws = torch.rand(n // 128, k // 128, device=DEV) + 0.5
    want = []
    for a in srcs:
        q = ops.quant_fp8(a)[0].clone()
        torch.cuda.synchronize()
        want.append(ops.linear_fp8(x, (q, ws)))
    torch.cuda.synchronize()
    g, out = torch.cuda.CUDAGraph(), []
    with torch.cuda.graph(g):
        for a in srcs * 4:
            # the last written values overwrite those of the call before in the same memory
            q = ops.quant_fp8(a)[0]
            out.append(ops.linear_fp8(x, (q, ws)))
            del q
    for _ in range(5):
        g.replay()
    torch.cuda.synchronize()
    for i, y in enumerate(out):
        assert torch.equal(y, want[i % 3]), i


def test_first_call_of_a_process_inside_a_capture():
    """Nothing that a first call sets up (attributes, cached sizes) is refused while a stream is captured."""
    import subprocess
    import sys
    code = """
import torch
from nanovllm_self_b200.ops import get_ops, torch_ref as R
ops = get_ops("cuda")
x = torch.randn(200, 512, device="cuda").bfloat16()
r0 = torch.randn(200, 512, device="cuda").bfloat16()
w = R.quant_fp8_weight(torch.randn(512, 512, device="cuda"))
one = torch.ones(512, device="cuda").bfloat16()
r = r0.clone()
torch.cuda.synchronize()
def step():
    h, _ = ops.add_rmsnorm_fp8(x, r, one, 1e-6)
    a = ops.linear_silu_fp8(h, w, 256)
    few = ops.quant_fp8(x[:5])
    return a[0].float(), ops.linear_fp8(h, w), ops.linear_fp8(few, w), ops.linear_silu_fp8(few, w, 256)[0].float()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    y = step()
g.replay()
torch.cuda.synchronize()
r.copy_(r0)
assert all(torch.equal(a, b) for a, b in zip(y, step()))
"""
    done = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=120)
    assert done.returncode == 0, done.stderr[-2000:]


def test_norm_of_the_residual_itself(ops):
    """x and the residual may be the same tensor: every value is read before it is written."""
    x, w = _acts(37, 1040), torch.ones(1040, device=DEV, dtype=torch.bfloat16)
    want = ops.add_rmsnorm_fp8(x, x.clone(), w, 1e-6)
    got = ops.add_rmsnorm_fp8(x, x, w, 1e-6)
    assert torch.equal(got[1], want[1])
    _same_pair(got[0], want[0])


# --------------------------------------------------------------------------- far offsets
def _wide_fp8(n, k):
    """[n, k] of e4m3 values, the bytes a cheap pattern without NaN."""
    q = torch.empty(n, k, dtype=torch.uint8, device=DEV)
    q.copy_((torch.arange(n, device=DEV) % 89)[:, None].to(torch.uint8))
    q += (torch.arange(k, device=DEV) % 23).to(torch.uint8)
    return q.view(torch.float8_e4m3fn)


@pytest.mark.parametrize("t,k", [(262153, 16), (600001, 32), (524321, 4112)])
def test_quant_and_norm_of_many_rows(ops, t, k):
    """More rows than one dimension of a grid holds CTAs, and (the last) offsets past 2^31 values."""
    x = torch.empty(t, k, dtype=torch.bfloat16, device=DEV)
    x.copy_(((torch.arange(t, device=DEV) % 509) + 1)[:, None])
    x *= ((torch.arange(k, device=DEV) % 7) - 3).to(torch.bfloat16)
    w = torch.ones(k, device=DEV, dtype=torch.bfloat16)
    for f in (ops.quant_fp8, lambda v: ops.add_rmsnorm_fp8(v, None, w, 1e-6)[0]):
        got = f(x)
        for rows in (slice(0, 40), slice(262140, 262153), slice(t - 33, t)):
            _same_pair((got[0][rows], got[1][rows]), f(x[rows]))


@pytest.mark.parametrize("t", [3, 200])
def test_products_of_weights_past_2_gib(ops, t):
    n, k = 524288 + 140, 4112
    q = _wide_fp8(n, k)
    s = torch.rand(-(-n // 128), -(-k // 128), device=DEV) + 0.5
    x = ops.quant_fp8(_acts(t, k))
    y = ops.linear_fp8(x, (q, s))
    for a, b in ((0, 256), (n // 128 * 128 - 256, n)):    # whole blocks of rows, the last ones among them
        part = (q[a:b], s[a // 128:-(-b // 128)])
        want = _exact(x, part)
        assert ((y[:, a:b].double() - want).abs() <= want.abs() * 2.0 ** -8 + 1.01 * _acc(k) * _bound(x, part)).all()


@pytest.mark.parametrize("t,n,act", [(131200, 16640, False), (131200, 33280, True)])
def test_products_with_outputs_past_2_gib(ops, t, n, act):
    k = 32
    x, w = ops.quant_fp8(_acts(t, k)), _weight(n, k)
    rows = slice(t - 70, t)
    few = ops.quant_fp8(_acts(t, k)[rows])
    if act:
        q, s = ops.linear_silu_fp8(x, w, n // 2)
        want = ops.linear_silu_fp8(few, w, n // 2)
        _same_pair((q[rows], s[rows]), want)
    else:
        want = _exact(few, w)
        y = ops.linear_fp8(x, w)[rows]
        assert ((y.double() - want).abs() <= want.abs() * 2.0 ** -8 + 1.01 * _acc(k) * _bound(few, w)).all()


# --------------------------------------------------------------------------- engine
def _llm(**kw):
    from nanovllm_self_b200 import LLM
    base = dict(device="cuda", max_model_len=1024, max_num_seqs=16, num_blocks=128, block_size=16, cuda_graph_max_bs=16,
                weight_quant_mode="fp8")
    base.update(kw)
    return LLM("tiny-gpu", **base)


def _prompts():
    g = torch.Generator().manual_seed(1)
    return [torch.randint(0, 2048, (n,), generator=g).tolist() for n in (17, 40, 64, 100)]


@pytest.mark.parametrize("kv", ["none", "fp8"])
def test_engine_logits_match_dense_oracle(kv):
    from nanovllm_self_b200 import SamplingParams
    from nanovllm_self_b200.engine.sequence import Sequence
    from nanovllm_self_b200.models.reference import dense_logits
    llm = _llm(kv_cache_quant_mode=kv)
    r = llm.model_runner
    for p in _prompts():
        s = Sequence(0, p, SamplingParams(temperature=0, max_tokens=1), r.block_size)
        r.block_manager.allocate(s)
        s.num_new_tokens = len(p) - s.num_cached_tokens
        got = r.logits([s])[0].float()
        r.block_manager.deallocate(s)
        ref = dense_logits(r.model, p)
        cos = torch.nn.functional.cosine_similarity(got, ref, dim=0).item()
        # The two differ by bf16 roundings, 2^-9 of a value, ahead of each rounding to e4m3, whose steps
        # are 2^-3: one value in 2^-3 / 2^-9 = 2^6 moves by a step, so an operand carries noise of
        # 2^-3 * sqrt(2^-6) = 2^-6 of itself, and each of the 8 products of the two layers adds as much:
        # sqrt(8) * 2^-6 = 0.044 of the logits, twice that with a margin, cos = 1 - 0.088^2 / 2 = 0.996.
        # The 8-bit cache's own noise (0.1, cos 0.995) adds in square: 1 - (0.088^2 + 0.1^2) / 2 = 0.991.
        assert cos > (0.996 if kv == "none" else 0.991), cos


def test_engine_graph_equals_eager():
    from nanovllm_self_b200 import SamplingParams
    sp = SamplingParams(temperature=0, max_tokens=16, ignore_eos=True)
    out = [_llm(enforce_eager=e).generate(_prompts(), sp) for e in (False, True)]
    assert out[0] == out[1]


@pytest.mark.parametrize("eager", [True, False])
def test_engine_reports_an_expired_wait(eager):
    """A bounded wait that runs out on the GPU reaches the caller of the engine, and only until it is reset."""
    from nanovllm_self_b200 import SamplingParams
    from nanovllm_self_b200.ops._ext import load
    C = load()
    llm = _llm(enforce_eager=eager)
    sp = SamplingParams(temperature=0, max_tokens=4, ignore_eos=True)
    want = llm.generate(_prompts(), sp)
    C.fp8_wait_check(1000000)     # nothing ends this wait: given up after a millisecond
    torch.cuda.synchronize()
    assert C.fp8_error() == 599
    with pytest.raises(RuntimeError, match="code 599"):
        llm.generate(_prompts(), sp)
    assert C.fp8_error(True) == 599 and C.fp8_error() == 0
    assert _llm(enforce_eager=eager).generate(_prompts(), sp) == want
