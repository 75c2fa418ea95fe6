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
    # |d silu| <= 1.1 |d gate|, silu <= |gate|; expf, a division and a product: 8 units
    err = 1.01 * _acc(k) * (1.1 * gb * up.abs() + gate.abs() * ub) + 8 * U * h.abs()
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
    for np_ in (16, 32, 64):
        if np_ >= t:
            for splits in (1, 2, 3, 4) if act else (1, 2, 3, 5, 8):
                yield [np_, splits]
    for splits in (1, 2, 4, 8):
        yield [0, splits]


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
    q0, s0 = C.linear_silu_fp8(*x, *w, i, [0, 1])
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
    for plan in ([16, 1], [32, 9], [128, 1], [24, 1], [32, 0], [32], [0, 3], [0, 16], [0, 0]):
        with pytest.raises(RuntimeError):
            ops.C.linear_fp8(*x, *w, None, plan)
    with pytest.raises(RuntimeError):
        ops.C.linear_silu_fp8(*x, *w, 128, [32, 5])


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
