"""The fp8 (e4m3) operators of the decoder layer, as they are measured.

One decoder layer of a model served with 8-bit weights runs, in this order: residual add + RMS norm
with an 8-bit output (``add_rmsnorm_fp8``), the q/k/v product (``linear_fp8``), attention, the 8-bit
form of the attention output (``quant_fp8``), the output product (``linear_fp8``), the norm again,
the gate/up product with SiLU-and-mul and an 8-bit output (``linear_silu_fp8``) and the down product
(``linear_fp8``).  Activations carry one fp32 scale per token and 128 channels, weights one per
block of 128 x 128.

``run`` computes an operator in its plain form (fp32 torch operations), or, with ``own`` set, by the
framework's kernels; ``exact`` computes the same from the definition in 64 bits.
"""
import math

import torch

own = False

G = 128            # channels of one scale
E4M3_MAX = 448.0
AMAX_MIN = 1e-30   # a group of zeros has the scale of this
EPS = 1e-6

_ops = None


def _framework():
    global _ops
    if _ops is None:
        from nanovllm_self_b200.ops import get_ops
        _ops = get_ops("cuda")
    return _ops


# ------------------------------------------------------------------------------------- cases
def listed():
    return [
        # the attention output of one decode token (Qwen3-8B): launch latency
        {"name": "quant 1x4096", "op": "quant", "t": 1, "k": 4096},
        # the attention outputs of a full prefill step (max_num_batched_tokens)
        {"name": "quant 16384x4096", "op": "quant", "t": 16384, "k": 4096},
        # a decode step at the benchmark's batch
        {"name": "norm 256x4096", "op": "norm", "t": 256, "k": 4096},
        # a ragged prefill step of Qwen3-32B
        {"name": "norm 8191x5120", "op": "norm", "t": 8191, "k": 5120},
        # q/k/v of one decode token
        {"name": "linear 1x6144x4096", "op": "linear", "t": 1, "n": 6144, "k": 4096},
        # down projection of a small batch
        {"name": "linear 17x4096x12288", "op": "linear", "t": 17, "n": 4096, "k": 12288},
        # output projection at the benchmark's batch
        {"name": "linear 256x4096x4096", "op": "linear", "t": 256, "n": 4096, "k": 4096},
        # a tensor-parallel shard with ragged sizes, a middling prompt
        {"name": "linear 1000x2744x1712", "op": "linear", "t": 1000, "n": 2744, "k": 1712},
        # down projection of a prefill step
        {"name": "linear 8192x4096x12288", "op": "linear", "t": 8192, "n": 4096, "k": 12288},
        # gate/up of one decode token
        {"name": "silu 1x12288x4096", "op": "silu", "t": 1, "n": 12288, "k": 4096},
        # gate/up at the benchmark's batch
        {"name": "silu 256x12288x4096", "op": "silu", "t": 256, "n": 12288, "k": 4096},
        # gate/up of a full prefill step
        {"name": "silu 16384x12288x4096", "op": "silu", "t": 16384, "n": 12288, "k": 4096},
    ]


def _log_int(rng, lo, hi, step=1):
    """An integer spread over the logarithm of [lo, hi], a multiple of ``step``."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(lo, min(hi, int(round(v / step)) * step))


def draw(rng):
    op = rng.choice(["quant", "norm", "linear", "linear", "silu"])
    t = _log_int(rng, 1, 16384)
    if op == "quant":
        return {"op": op, "t": t, "k": _log_int(rng, 64, 25600, 16)}
    if op == "norm":
        return {"op": op, "t": t, "k": _log_int(rng, 64, 8192, 16)}
    k = _log_int(rng, 64, 12288, 16)
    # outputs of any width (vocabulary and tensor-parallel shards are not always round); products
    # no larger than the largest listed one
    n = _log_int(rng, 64, 12288, 1 if op == "linear" else 16)
    return {"op": op, "t": min(t, 800_000_000_000 // (n * k)), "n": n, "k": k}


def work(case):
    t, k = case["t"], case["k"]
    kb = -(-k // G)
    if case["op"] == "quant":
        return {"bytes": 2 * t * k + t * k + 4 * t * kb, "flops": 3 * t * k}
    if case["op"] == "norm":
        return {"bytes": 4 * t * k + 2 * k + 2 * t * k + t * k + 4 * t * kb, "flops": 8 * t * k}
    n = case["n"]
    nb = -(-n // G)
    if case["op"] == "linear":
        return {"bytes": t * k + 4 * t * kb + n * k + 4 * nb * kb + 2 * t * n, "flops": 2 * t * n * k}
    return {"bytes": t * k + 4 * t * kb + 2 * n * k + 8 * nb * kb + t * n + 4 * t * nb, "flops": 4 * t * n * k}


# ------------------------------------------------------------------------------------- inputs
def _activations(t, k, gen):
    """Normal values whose channels differ in size, a few of them by far (as a decoder's do)."""
    x = torch.randn(t, k, device="cuda", generator=gen)
    c = torch.exp(0.5 * torch.randn(k, device="cuda", generator=gen))
    c = torch.where(torch.rand(k, device="cuda", generator=gen) < 0.002, 20.0 * c, c)
    return (x * c).to(torch.bfloat16)


def _weight(n, k, gen, pad_to=None):
    """N(0, 0.02) weights [n, k] as e4m3 with one scale per block of 128 x 128; rows up to
    ``pad_to`` are zero."""
    w = 0.02 * torch.randn(n, k, device="cuda", generator=gen)
    if pad_to is not None and pad_to > n:
        w = torch.cat([w, w.new_zeros(pad_to - n, k)])
    return w


def _quant_weight(w):
    n, k = w.shape
    nb, kb = -(-n // G), -(-k // G)
    p = w.new_zeros(nb * G, kb * G)
    p[:n, :k] = w
    p = p.view(nb, G, kb, G)
    a = p.abs().amax(dim=(1, 3)).clamp(min=AMAX_MIN)
    q = (p * (E4M3_MAX / a)[:, None, :, None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
    return q.view(nb * G, kb * G)[:n, :k].contiguous(), a / E4M3_MAX


def _token_contiguous(s):
    """The layout the framework keeps activation scales in: [T, K / 128] with unit stride over the
    tokens and a column stride that is a multiple of 4."""
    t, kb = s.shape
    buf = s.new_zeros(kb, -(-t // 4) * 4)
    buf[:, :t] = s.t()
    return buf[:, :t].t()


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    t, k, op = case["t"], case["k"], case["op"]
    st = {"op": op, "x": _activations(t, k, gen)}
    if op == "norm":
        st["residual"] = (3.0 * torch.randn(t, k, device="cuda", generator=gen)).to(torch.bfloat16)
        st["w"] = (1.0 + 0.2 * torch.randn(k, device="cuda", generator=gen)).to(torch.bfloat16)
    elif op in ("linear", "silu"):
        q, s = _quant(st.pop("x").float())
        st["xq"], st["xs"] = q, _token_contiguous(s)
        n = case["n"]
        if op == "linear":
            st["wq"], st["ws"] = _quant_weight(_weight(n, k, gen))
        else:
            ib = -(-n // G)
            gate, up = (_weight(n, k, gen, ib * G).view(ib, 1, G, k) for _ in range(2))
            # blocks of 128 gate rows and the 128 matching up rows in turn
            st["wq"], st["ws"] = _quant_weight(torch.cat([gate, up], 1).reshape(2 * ib * G, k))
            st["features"] = n
    return st


# ------------------------------------------------------------------------------------- plain form
def _quant(x):
    """x [T, K] fp32 -> (e4m3 values [T, K], scales [T, ceil(K / 128)])."""
    t, k = x.shape
    kb = -(-k // G)
    if kb * G != k:
        p = x.new_zeros(t, kb * G)
        p[:, :k] = x
        x = p
    x = x.view(t, kb, G)
    a = x.abs().amax(-1).clamp(min=AMAX_MIN)
    q = (x * (E4M3_MAX / a)[..., None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
    return q.view(t, kb * G)[:, :k].contiguous(), a / E4M3_MAX


def _product(xq, xs, wq, ws):
    """fp32 [T, N] of the dequantised operands."""
    k, n = xq.shape[1], wq.shape[0]
    x = xq.float() * xs.repeat_interleave(G, 1)[:, :k]
    w = wq.float() * ws.repeat_interleave(G, 0)[:n].repeat_interleave(G, 1)[:, :k]
    return x @ w.t()


def run(state):
    op = state["op"]
    if own:
        ops = _framework()
        if op == "quant":
            return ops.quant_fp8(state["x"])
        if op == "norm":
            return ops.add_rmsnorm_fp8(state["x"], state["residual"], state["w"], EPS)
        x, w = (state["xq"], state["xs"]), (state["wq"], state["ws"])
        if op == "linear":
            return ops.linear_fp8(x, w)
        return ops.linear_silu_fp8(x, w, state["features"])
    if op == "quant":
        return _quant(state["x"].float())
    if op == "norm":
        # the residual stream is updated in place, as the model's norm does
        r = state["residual"].copy_(state["x"].float() + state["residual"].float())
        f = r.float()
        y = f * torch.rsqrt(f.square().mean(-1, keepdim=True) + EPS) * state["w"].float()
        return _quant(y), r
    y = _product(state["xq"], state["xs"], state["wq"], state["ws"])
    if op == "linear":
        return y.to(torch.bfloat16)
    t, n = y.shape
    y = y.view(t, n // (2 * G), 2, G)
    g, u = y[:, :, 0], y[:, :, 1]
    h = g / (1.0 + torch.exp(-g)) * u
    return _quant(h.reshape(t, n // 2)[:, :state["features"]])


# ------------------------------------------------------------------------------------- 64 bits
def _e4m3_64(v):
    """Nearest e4m3 value of a float64 (ties to the even mantissa, beyond the range the largest)."""
    v = v.clamp(-448.0, 448.0)
    e = torch.frexp(v.abs())[1].to(torch.float64) - 1.0
    step = torch.exp2(e.clamp(min=-6.0) - 3.0)
    return (torch.round(v / step) * step).clamp(-448.0, 448.0)


def _quant_64(y):
    k = y.shape[1]
    cols = torch.arange(k, device=y.device) // 128
    amax = torch.full((y.shape[0], (k + 127) // 128), 1e-30, dtype=torch.float64, device=y.device)
    amax = amax.scatter_reduce(1, cols.expand_as(y), y.abs(), "amax")
    return _e4m3_64(y * (448.0 / amax)[:, cols]), amax / 448.0


def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op == "quant":
        return _quant_64(st["x"].double())
    if op == "norm":
        r = (st["x"].double() + st["residual"].double()).to(torch.bfloat16).double()
        y = r / torch.sqrt((r * r).sum(1, keepdim=True) / r.shape[1] + EPS) * st["w"].double()
        return _quant_64(y), r
    k, n = st["xq"].shape[1], st["wq"].shape[0]
    kb = torch.arange(k, device="cuda") // 128
    nb = torch.arange(n, device="cuda") // 128
    x = st["xq"].double() * st["xs"].double()[:, kb]
    w = st["wq"].double() * st["ws"].double()[nb][:, kb]
    y = torch.einsum("tk,nk->tn", x, w)
    del x, w
    if op == "linear":
        return y
    f = torch.arange(case["n"], device="cuda")
    row = f // 128 * 256 + f % 128
    g, u = y[:, row], y[:, row + 128]
    del y
    return _quant_64(g * torch.sigmoid(g) * u)
