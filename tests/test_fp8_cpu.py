"""fp8 weights and activations on CPU: the block formats, the engine on them, and the kernels' refusals."""
import pytest
import torch

from nanovllm_self_b200 import LLM, SamplingParams
from nanovllm_self_b200.config import EngineConfig
from nanovllm_self_b200.models.configs import Qwen3Arch
from nanovllm_self_b200.models.loader import random_init
from nanovllm_self_b200.models.qwen3 import Qwen3ForCausalLM
from nanovllm_self_b200.models.reference import dense_logits, greedy_generate
from nanovllm_self_b200.ops import get_ops, torch_ref as R


# --------------------------------------------------------------------------- formats
@pytest.mark.parametrize("t,k", [(1, 16), (3, 128), (5, 272), (2, 4096)])
def test_quant_rounds_within_half_a_step(t, k):
    x = torch.randn(t, k, generator=torch.Generator().manual_seed(k)) * torch.logspace(-3, 2, k)
    q, s = R.quant_fp8(x)
    assert q.dtype == torch.float8_e4m3fn and s.shape == (t, -(-k // 128))
    d, sc = R.dequant_fp8(q, s, torch.float64), s.double().repeat_interleave(128, 1)[:, :k]
    # half a step of e4m3 is 2^-4 of the value, or 2^-10 of the scale; fp32 arithmetic adds 4 units
    assert ((d - x.double()).abs() <= x.double().abs() * (2.0 ** -4 + 2.0 ** -21) + sc * 2.0 ** -10 * (1 + 2.0 ** -21)).all()
    full = x[:, :k // 128 * 128]
    if full.numel():  # the largest magnitude of a group maps to 448
        assert (q[:, :full.shape[1]].float().view(t, -1, 128).abs().amax(-1) == 448).all()


def test_quant_weight_blocks_and_padding_of_gate_up():
    g = torch.Generator().manual_seed(1)
    w = torch.randn(300, 200, generator=g)
    w[128:256, :128] = 0
    q, s = R.quant_fp8_weight(w)
    assert q.shape == w.shape and s.shape == (3, 2)
    assert s[1, 0] == torch.tensor(R.FP8_AMAX_MIN) / 448 and (R.dequant_fp8_weight(q, s)[128:256, :128] == 0).all()
    assert s[2, 1] == w[256:, 128:].abs().max() / 448
    gate, up = torch.randn(200, 48, generator=g), torch.randn(200, 48, generator=g)
    gu = R.group_gate_up(gate, up)
    assert gu.shape == (512, 48)
    assert torch.equal(gu[:128], gate[:128]) and torch.equal(gu[128:256], up[:128])
    assert torch.equal(gu[256:328], gate[128:]) and torch.equal(gu[384:456], up[128:])
    assert (gu[328:384] == 0).all() and (gu[456:] == 0).all()


def test_products_match_dequantised_operands():
    g = torch.Generator().manual_seed(2)
    ops = get_ops("cpu")
    x = ops.quant_fp8(torch.randn(7, 272, generator=g))
    w = R.quant_fp8_weight(torch.randn(130, 272, generator=g))
    want = R.dequant_fp8(*x, torch.float64) @ R.dequant_fp8_weight(*w, torch.float64).t()
    got = ops.linear_fp8(x, w, dtype=torch.float32)
    assert ((got.double() - want).abs() <= 272 * 2.0 ** -22 * want.abs().max()).all()
    out = torch.empty(7, 130)
    assert ops.linear_fp8(x, w, out=out) is out and torch.equal(out, got)
    gate, up = torch.randn(144, 272, generator=g) / 16, torch.randn(144, 272, generator=g) / 16
    gu = R.quant_fp8_weight(R.group_gate_up(gate, up))
    q, s = ops.linear_silu_fp8(x, gu, 144)
    assert q.shape == (7, 144) and s.shape == (7, 2)
    y = R.dequant_fp8(*x, torch.float64) @ R.dequant_fp8_weight(*gu, torch.float64).t()
    a, b = torch.cat([y[:, :128], y[:, 256:272]], 1), torch.cat([y[:, 128:256], y[:, 384:400]], 1)
    h = a * torch.sigmoid(a) * b
    sc = s.double().repeat_interleave(128, 1)[:, :144]
    assert ((q.double() * sc - h).abs() <= h.abs() * (2.0 ** -4 + 2.0 ** -16) + sc * 2.0 ** -10 * 1.001).all()


# --------------------------------------------------------------------------- engine
def _llm(**kw):
    base = dict(device="cpu", dtype="fp32", block_size=16, max_model_len=512, num_blocks=128,
                weight_quant_mode="fp8")
    base.update(kw)
    return LLM("tiny", **base)


def _prompts():
    g = torch.Generator().manual_seed(0)
    return [torch.randint(0, 1024, (n,), generator=g).tolist() for n in (16, 33, 48)]


def test_engine_on_fp8_weights_equals_its_dense_oracle():
    llm = _llm()
    m = llm.model_runner.model
    L = m.layers[0]
    for q, s in (L.qkv, L.o, L.gate_up, L.down):
        assert q.dtype == torch.float8_e4m3fn and s.dtype == torch.float32
    out = llm.generate(_prompts(), SamplingParams(temperature=0, max_tokens=8, ignore_eos=True))
    for p, o in zip(_prompts(), out):
        assert o[len(p):] == greedy_generate(m, p, 8)


def test_fp8_weights_stay_near_the_full_precision_model_and_take_fewer_bytes():
    a, b = _llm(), _llm(weight_quant_mode="none")
    p = _prompts()[1]
    x, y = dense_logits(a.model_runner.model, p), dense_logits(b.model_runner.model, p)
    # every operand of the products moves by up to 2^-4 of itself, about 2^-5.3 on average; independent
    # roundings average out over the sums
    assert torch.nn.functional.cosine_similarity(x, y, dim=0) > 0.99
    ma, mb = a.model_runner.model, b.model_runner.model
    assert ma.weight_bytes() < mb.weight_bytes()


def test_chunked_prefill_and_bf16_model_run_on_fp8_weights():
    out = _llm(enable_chunked_prefill=True, prefill_chunk_size=20, max_num_batched_tokens=40, dtype="bf16").generate(
        _prompts(), SamplingParams(temperature=0, max_tokens=4, ignore_eos=True))
    assert [len(o) for o in out] == [len(p) + 4 for p in _prompts()]


def test_engine_returns_no_token_of_a_product_that_gave_up(monkeypatch):
    llm = _llm()
    sp = SamplingParams(temperature=0, max_tokens=4, ignore_eos=True)
    llm.generate(_prompts(), sp)
    monkeypatch.setattr(llm.model_runner.ops, "device_error", lambda: 501)
    for _ in range(2):   # it stays: the KV cache may hold what came of it
        with pytest.raises(RuntimeError, match="bounded wait .code 501"):
            llm.generate(_prompts(), sp)
    other = _llm(weight_quant_mode="none")   # runs no fp8 product
    assert other.model_runner.ops.device_error() == 501
    assert [len(o) for o in other.generate(_prompts(), sp)] == [len(p) + 4 for p in _prompts()]


ARCH = Qwen3Arch(vocab_size=256, hidden_size=128, intermediate_size=512, num_hidden_layers=1, num_attention_heads=4,
                 num_key_value_heads=2, head_dim=128, max_position_embeddings=256, tie_word_embeddings=False)


def test_tensor_parallel_shards_hold_the_same_blocks():
    """Where a rank's shares are whole blocks of 128, sharding does not change the quantised weights."""
    whole = random_init(Qwen3ForCausalLM(ARCH, dtype=torch.float32, weight_quant="fp8")).layers[0]
    bits = lambda t: t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t  # noqa: E731
    for r in range(2):
        L = random_init(Qwen3ForCausalLM(ARCH, r, 2, dtype=torch.float32, weight_quant="fp8")).layers[0]
        for i, unit in ((0, 128), (1, 1)):  # values, scales
            q, k, v = (bits(whole.qkv[i])[a * unit:b * unit] for a, b in ((0, 4), (4, 6), (6, 8)))
            want = torch.cat([t[r * n * unit:(r + 1) * n * unit] for t, n in ((q, 2), (k, 1), (v, 1))])
            assert torch.equal(bits(L.qkv[i]), want)
            assert torch.equal(bits(L.o[i]), bits(whole.o[i])[:, 2 * unit * r:2 * unit * (r + 1)])
            assert torch.equal(bits(L.gate_up[i]), bits(whole.gate_up[i])[4 * unit * r:4 * unit * (r + 1)])
            assert torch.equal(bits(L.down[i]), bits(whole.down[i])[:, 2 * unit * r:2 * unit * (r + 1)])


def _tp_worker(rank, world, port, path):
    import json
    import os
    import torch.distributed as dist
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port), RANK=str(rank), WORLD_SIZE=str(world),
                      LOCAL_RANK=str(rank))
    out = LLM("tiny-gpu", tensor_parallel_size=world, **_tp_kw()).generate(
        _prompts(), SamplingParams(temperature=0, max_tokens=8, ignore_eos=True))
    with open(f"{path}.{rank}", "w") as f:
        json.dump(out, f)
    dist.barrier()
    os._exit(0)  # no teardown of the gloo group: its destructor can race with its own threads at exit


def _tp_kw():
    return dict(device="cpu", dtype="fp32", block_size=16, max_model_len=256, num_blocks=64, comm_backend="nccl",
                weight_quant_mode="fp8")


def test_tensor_parallel_engine_equals_one_rank(tmp_path):
    import json
    import socket
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    path = str(tmp_path / "tp")
    torch.multiprocessing.spawn(_tp_worker, args=(2, port, path), nprocs=2, join=True)
    outs = [json.load(open(f"{path}.{r}")) for r in range(2)]
    want = LLM("tiny-gpu", **_tp_kw()).generate(_prompts(), SamplingParams(temperature=0, max_tokens=8, ignore_eos=True))
    assert outs[0] == outs[1] == want


# --------------------------------------------------------------------------- refusals
def test_config_refusals():
    with pytest.raises(ValueError, match="weight_quant_mode"):
        EngineConfig(weight_quant_mode="int4")
    with pytest.raises(ValueError, match="bf16"):
        EngineConfig(weight_quant_mode="fp8", dtype="fp16")
    with pytest.raises(ValueError, match="fused_reduce_scatter"):
        EngineConfig(weight_quant_mode="fp8", fused_reduce_scatter=True)
    bad = Qwen3Arch(vocab_size=64, hidden_size=40, intermediate_size=64, num_hidden_layers=1, num_attention_heads=2,
                    num_key_value_heads=1, head_dim=32)
    with pytest.raises(ValueError, match="multiple of 16"):
        Qwen3ForCausalLM(bad, weight_quant="fp8")


@pytest.fixture(scope="module")
def C():
    ext = pytest.importorskip("nanovllm_self_b200._C")
    return ext


def _x(t=4, k=256, dtype=torch.bfloat16):
    return torch.zeros(t, k, dtype=dtype)


def _refused(f, match):
    with pytest.raises(RuntimeError, match=match):
        f()


def test_quant_and_norm_refusals(C):
    _refused(lambda: C.quant_fp8(_x()), "CUDA")                                  # everything else is fine
    _refused(lambda: C.quant_fp8(_x(dtype=torch.float16)), "bfloat16")
    _refused(lambda: C.quant_fp8(_x(k=40)), "multiple of 16")
    _refused(lambda: C.quant_fp8(_x(k=0)), "multiple of 16")
    _refused(lambda: C.quant_fp8(_x()[0]), "unit inner stride")
    _refused(lambda: C.quant_fp8(_x(256, 256).t()), "unit inner stride")
    _refused(lambda: C.quant_fp8(_x(4, 260)[:, :256]), "row stride")
    _refused(lambda: C.quant_fp8(_x(1, 256).expand(4, 256)), "row stride")
    _refused(lambda: C.quant_fp8(_x(4, 512)[:, 4:260]), "aligned")
    w = torch.ones(256, dtype=torch.bfloat16)
    _refused(lambda: C.add_rmsnorm_fp8(_x(), None, w, 1e-6), "CUDA")
    _refused(lambda: C.add_rmsnorm_fp8(_x(), _x(), w, 1e-6), "CUDA")
    _refused(lambda: C.add_rmsnorm_fp8(_x(), None, w[:128], 1e-6), "256 contiguous")
    _refused(lambda: C.add_rmsnorm_fp8(_x(), None, w.float(), 1e-6), "256 contiguous")
    _refused(lambda: C.add_rmsnorm_fp8(_x(), _x(3), w, 1e-6), "residual")
    _refused(lambda: C.add_rmsnorm_fp8(_x(), _x(4, 512)[:, :256], w, 1e-6), "residual")
    _refused(lambda: C.add_rmsnorm_fp8(_x(), _x(dtype=torch.float32), w, 1e-6), "residual")
    _refused(lambda: C.add_rmsnorm_fp8(_x(1, 16400), None, torch.ones(16400, dtype=torch.bfloat16), 1e-6), "16384")


def test_residual_over_other_rows_of_x_is_refused(C):
    """Rows are read and written in any order: a residual over another row's input is not defined."""
    w = torch.ones(256, dtype=torch.bfloat16)
    big = _x(10, 256)
    _refused(lambda: C.add_rmsnorm_fp8(big[:4], big[:4], w, 1e-6), "CUDA")     # the same rows: in place
    _refused(lambda: C.add_rmsnorm_fp8(big[:4], big[4:8], w, 1e-6), "CUDA")
    _refused(lambda: C.add_rmsnorm_fp8(big[1:5], big[:4], w, 1e-6), "in common")
    _refused(lambda: C.add_rmsnorm_fp8(big[:8:2], big[:4], w, 1e-6), "in common")
    _refused(lambda: C.add_rmsnorm_fp8(_x(), big[:4], big[2], 1e-6), "in common")
    _refused(lambda: C.add_rmsnorm_fp8(big[::8], big[1:3], w, 1e-6), "CUDA")   # between x's rows
    # against every element's address, over all places of a few shapes
    store = torch.zeros(64 * 16, dtype=torch.bfloat16)
    at = store.data_ptr()
    for t, ld in ((1, 16), (2, 16), (2, 48), (3, 24), (4, 64)):
        x = store[16 * 20:].as_strided((t, 16), (ld, 1))
        mine = {x.data_ptr() + 2 * (i * ld + j) for i in range(t) for j in range(16)}
        for off in range(0, 64 * 16 - 16 * t, 8):
            r = store[off:off + 16 * t].view(t, 16)
            meets = any(at + 2 * (off + j) in mine for j in range(16 * t))
            same = r.data_ptr() == x.data_ptr() and (ld == 16 or t == 1)
            _refused(lambda: C.add_rmsnorm_fp8(x, r, w[:16], 1e-6), "in common" if meets and not same else "CUDA")


def test_messages_hold_numbers_and_shapes(C):
    """In a process of its own: with a second copy of the C++ library in the extension a number in a message ends
    the process."""
    import subprocess
    import sys
    code = """
import torch
from nanovllm_self_b200.ops._ext import load
C = load()
f8 = torch.float8_e4m3fn
def message(f):
    try:
        f()
    except RuntimeError as e:
        return str(e)
print(message(lambda: C.quant_fp8(torch.zeros(4, 40, dtype=torch.bfloat16))))
xs = torch.zeros(2, 8)[:, :6].t()
print(message(lambda: C.linear_fp8(torch.zeros(6, 256).to(f8), xs, torch.zeros(256, 240).to(f8), torch.zeros(2, 2))))
"""
    done = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=120)
    assert done.returncode == 0, (done.returncode, done.stderr[-500:])
    assert "multiple of 16, got 40" in done.stdout and "[6, 256] and [256, 240]" in done.stdout
    with open(C.__file__, "rb") as f:
        assert b"\0libstdc++.so.6\0" in f.read()   # linked to the library that torch uses


def test_sizes_that_do_not_fit_the_kernels_integers_are_refused(C):
    """2^32 + 128 channels would be taken for 128 of them."""
    for x in (torch.empty(0, 2 ** 32 + 128, dtype=torch.bfloat16), torch.empty(0, 2 ** 31, dtype=torch.bfloat16),
              torch.empty(2 ** 32 + 1, 16, dtype=torch.bfloat16, device="meta")):
        _refused(lambda: C.quant_fp8(x), "too large")


def _operands(t=6, n=256, k=256):
    f8 = torch.float8_e4m3fn
    xs = torch.zeros(-(-k // 128), 8)[:, :t].t()
    return [torch.zeros(t, k).to(f8), xs, torch.zeros(n, k).to(f8), torch.zeros(-(-n // 128), -(-k // 128))]


def test_product_refusals(C):
    def bad(i, v, match, f=C.linear_fp8, *more):
        a = _operands()
        a[i] = v
        _refused(lambda: f(*a, *more), match)

    f8 = torch.float8_e4m3fn
    _refused(lambda: C.linear_fp8(*_operands()), "CUDA")
    _refused(lambda: C.linear_silu_fp8(*_operands(), 128), "CUDA")
    bad(0, torch.zeros(6, 256, dtype=torch.bfloat16), "float8_e4m3fn")
    bad(2, torch.zeros(256, 256, dtype=torch.float8_e5m2), "float8_e4m3fn")
    bad(1, _operands()[1].half(), "float32")
    bad(2, torch.zeros(256, 240).to(f8), "multiple of 16")
    bad(0, torch.zeros(6, 264).to(f8)[:, :256], "multiples of 16")
    bad(0, torch.zeros(6, 272).to(f8)[:, 8:264], "aligned|alignment")
    bad(1, torch.zeros(6, 2), "token-contiguous")            # row-major scales
    bad(1, torch.zeros(2, 7)[:, :6].t(), "token-contiguous")  # a column stride that is no multiple of 4
    bad(1, torch.zeros(2, 8).t(), "scales must be")
    bad(3, torch.zeros(2, 3), "scales must be")
    bad(3, torch.zeros(2, 2).t().contiguous().t(), "scales must be")
    a = _operands()
    for out in (torch.zeros(6, 256), torch.zeros(5, 256, dtype=torch.bfloat16),
                torch.zeros(256, 6, dtype=torch.bfloat16).t()):
        _refused(lambda: C.linear_fp8(*a, out), "out must be")
    for features in (0, 120, 129, 64 * 1024):
        _refused(lambda: C.linear_silu_fp8(*a, features), "features")
    _refused(lambda: C.linear_silu_fp8(*a, 144), "features")  # w has one pair of blocks, not two


def test_plans_of_any_gpu_size_and_their_refusals(C):
    """In a process of its own: a plan for a GPU of no SMs, or one, divided by zero and ended the process."""
    import subprocess
    import sys
    code = """
from nanovllm_self_b200.ops._ext import load
C = load()
for sms in (1, 2, 3, 7, 148, 160):
    for t, n, k, act in ((0, 0, 16, 0), (1, 16, 16, 0), (33, 256, 1040, 1), (200, 4096, 4096, 0), (9000, 24576, 4096, 1)):
        np_, splits = C.fp8_plan(t, n, k, act, sms)
        assert np_ in (-1, -2, -3) or t <= np_ <= 64
        assert 1 <= splits <= 8
for bad in ((-1, 16, 16, 0, 148), (1, -16, 16, 0, 148), (1, 16, 0, 0, 148), (200, 256, 256, 0, 0), (200, 256, 256, 0, -4),
            (200, 256, 256, 2, 148), (2 ** 32 + 1, 256, 256, 0, 148), (1, 2 ** 33, 256, 0, 148), (1, 16, 2 ** 32 + 16, 0, 148)):
    try:
        C.fp8_plan(*bad)
    except RuntimeError:
        continue
    raise SystemExit(f"not refused: {bad}")
"""
    done = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=120)
    assert done.returncode == 0, (done.returncode, done.stderr[-500:])


@pytest.mark.parametrize("sizes,plan", [((1, 4480, 4096, 0), [16, 7]), ((1, 9216, 4096, 0), [16, 3]),
                                        ((1, 11904, 4096, 0), [16, 2]), ((1, 7040, 4096, 0), [16, 4]),
                                        ((1, 9216, 4096, 1), [16, 7]), ((256, 4096, 4096, 0), [-3, 2]),
                                        ((1024, 12288, 4096, 1), [-2, 1])])
def test_plan_without_a_gpu_is_that_of_a_b200(C, sizes, plan):
    """A plan fixes the order of the sums, so it must not depend on what the process can ask a GPU.  All
    but the last two lie just past what a B200 holds: 35 or 36 tiles in clusters of 8 (33), 72 of 4 (71), 93 of 3
    (92), 55 of 5 (53)."""
    assert C.fp8_plan(*sizes, 148) == plan


def test_every_slice_of_a_plan_has_work(C):
    for t in (1, 16, 17, 33, 64, 65, 130, 256, 500, 2000):
        for act in (0, 1):
            for kb in list(range(1, 70)) + [96, 100, 128, 200]:
                for n in (256, 768, 2048, 4608, 6144, 8960, 9216, 24576):
                    splits = C.fp8_plan(t, n, kb * 128, act, 148)[1]
                    per = -(-kb // splits)
                    assert (splits - 1) * per < kb, (t, n, kb, act, splits)
