"""The operators of the 8-bit path where no GPU is needed: the ABI, every refusal that comes before a launch, empty calls."""
import os
import re
import subprocess
import sys

import pytest
import torch

from codegendemo_amd import _native, _native_ops
from codegendemo_amd.kcg.Operators.matmul_fp8 import matmul_fp8
from codegendemo_amd.kcg.Operators.moe import moe_layer
from codegendemo_amd.kcg.Operators.quant import rmsnorm_quant, swiglu_quant

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BF16, F16, F32, F64, E4M3 = 3, 2, 4, 8, 1
P = 0x10000                                       # an address on 16 bytes that nothing is read from

STRUCTS = {"kcg_rmsnorm_quant": _native_ops.RMSNORM_QUANT, "kcg_swiglu_quant": _native_ops.SWIGLU_QUANT,
           "kcg_matmul_fp8": _native_ops.MATMUL_FP8, "kcg_moe_layer": _native_ops.MOE_LAYER}


def header():
    with open(os.path.join(ROOT, "include", "kcg_ops.h")) as f:
        return re.sub(r"/\*.*?\*/", "", f.read(), flags=re.S)


def fields(call):
    body = re.search(r"typedef struct %s_args \{(.*?)\}" % call, header(), flags=re.S).group(1)
    names = []
    for line in body.split(";"):
        line = line.strip()
        if line:
            names += [(n.strip(), line.split()[0]) for n in line.split(None, 1)[1].split(",")]
    return names


def test_every_declared_symbol_is_exported_and_bound():
    names = sorted(set(re.findall(r"\b(kcg_[a-z0-9_]+)\s*\(", header())))
    assert set(names) == set(_native_ops.EXPORTS)
    for n in names:
        assert hasattr(_native_ops.lib(), n)


@pytest.mark.parametrize("call", list(STRUCTS))
def test_packed_arguments_match_the_declared_struct(call):
    declared = fields(call)
    code = "".join("q" if t == "int64_t" else "d" for _, t in declared)
    packed = STRUCTS[call].format.lstrip("=")
    assert re.sub(r"(\d+)(\w)", lambda m: m.group(2) * int(m.group(1)), packed) == code


GOOD = {
    "kcg_rmsnorm_quant": dict(x=P, residual=P, residual_out=P, weight=P, y=P, q=P, scale=P, x_stride=256, residual_stride=256, residual_out_stride=256,
                              y_stride=256, q_stride=256, scale_stride_row=2, scale_stride_group=1, rows=4, cols=250, dtype=BF16, weight_dtype=F32, eps=1e-6),
    "kcg_swiglu_quant": dict(gate_up=P, q=P, scale=P, gate_up_stride=512, q_stride=256, scale_stride_row=2, scale_stride_group=1, rows=4, cols=250, dtype=F16),
    "kcg_matmul_fp8": dict(a=P, a_scale=P, b=P, b_scale=P, c=P, a_stride=208, a_scale_stride_row=2, a_scale_stride_group=1, b_stride=208,
                           b_scale_stride_row=2, b_scale_stride_group=1, c_stride=300, m=4, n=300, k=200, c_dtype=F32),
    "kcg_moe_layer": dict(x=P, logits=P, w13=P, w13_scale=P, w2=P, w2_scale=P, out=P, ids=P, probs=P, workspace=P, workspace_bytes=1 << 20, x_stride=64,
                          logits_stride=8, out_stride=64, w13_stride_expert=96 * 64, w13_stride_row=64, w2_stride_expert=64 * 48, w2_stride_row=48, tokens=3,
                          experts=8, topk=2, hidden=64, inter=48, dtype=BF16, weight_dtype=E4M3, renormalize=1),
}

BAD = [
    ("kcg_rmsnorm_quant", dict(dtype=F64), "bfloat16, float16 or float32"), ("kcg_rmsnorm_quant", dict(dtype=E4M3), "bfloat16, float16 or float32"),
    ("kcg_rmsnorm_quant", dict(weight_dtype=F16), "weight"), ("kcg_rmsnorm_quant", dict(rows=-1), "rows and cols"),
    ("kcg_rmsnorm_quant", dict(cols=(1 << 30) + 1), "rows and cols"), ("kcg_rmsnorm_quant", dict(eps=-1.0), "eps"), ("kcg_rmsnorm_quant", dict(eps=float("nan")), "eps"),
    ("kcg_rmsnorm_quant", dict(residual=0), "go together"), ("kcg_rmsnorm_quant", dict(residual_out=0), "go together"),
    ("kcg_rmsnorm_quant", dict(x=0), "null"), ("kcg_rmsnorm_quant", dict(weight=0), "null"), ("kcg_rmsnorm_quant", dict(q=0), "null"),
    ("kcg_rmsnorm_quant", dict(scale=0), "null"), ("kcg_rmsnorm_quant", dict(x=P + 1), "aligned"), ("kcg_rmsnorm_quant", dict(scale=P + 2), "aligned"),
    ("kcg_rmsnorm_quant", dict(weight=P + 2), "aligned"), ("kcg_rmsnorm_quant", dict(q=P + 8), "16 bytes"), ("kcg_rmsnorm_quant", dict(q_stride=250), "16 bytes"),
    ("kcg_rmsnorm_quant", dict(x_stride=-256), "row stride"), ("kcg_rmsnorm_quant", dict(q_stride=240), "row stride"), ("kcg_rmsnorm_quant", dict(y_stride=249), "row stride"),
    ("kcg_rmsnorm_quant", dict(residual_out_stride=0), "row stride"), ("kcg_rmsnorm_quant", dict(scale_stride_row=1), "overlap"),
    ("kcg_rmsnorm_quant", dict(scale_stride_group=0), "overlap"), ("kcg_rmsnorm_quant", dict(scale_stride_row=0), "overlap"),
    ("kcg_swiglu_quant", dict(dtype=F64), "bfloat16, float16 or float32"), ("kcg_swiglu_quant", dict(cols=-1), "rows and cols"), ("kcg_swiglu_quant", dict(gate_up=0), "null"),
    ("kcg_swiglu_quant", dict(gate_up=P + 1), "aligned"), ("kcg_swiglu_quant", dict(q=P + 4), "16 bytes"), ("kcg_swiglu_quant", dict(q_stride=248), "16 bytes"),
    ("kcg_swiglu_quant", dict(gate_up_stride=-1), "row stride"), ("kcg_swiglu_quant", dict(q_stride=16), "row stride"), ("kcg_swiglu_quant", dict(scale_stride_row=1), "overlap"),
    ("kcg_swiglu_quant", dict(rows=1 << 28, q_stride=256), "too large"), ("kcg_rmsnorm_quant", dict(rows=1 << 28), "too large"),
    ("kcg_matmul_fp8", dict(m=1 << 30, n=1 << 30, c_stride=1 << 30), "too large"),
    ("kcg_matmul_fp8", dict(c_dtype=F64), "bfloat16, float16 or float32"), ("kcg_matmul_fp8", dict(m=-1), "m, n and k"), ("kcg_matmul_fp8", dict(k=(1 << 30) + 1), "m, n and k"),
    ("kcg_matmul_fp8", dict(a=0), "null"), ("kcg_matmul_fp8", dict(b_scale=0), "null"), ("kcg_matmul_fp8", dict(c=0), "null"), ("kcg_matmul_fp8", dict(c=P + 2), "aligned"),
    ("kcg_matmul_fp8", dict(a_scale=P + 1), "aligned"), ("kcg_matmul_fp8", dict(a=P + 8), "16 bytes"), ("kcg_matmul_fp8", dict(b_stride=200), "16 bytes"),
    ("kcg_matmul_fp8", dict(a_stride=192), "row stride"), ("kcg_matmul_fp8", dict(c_stride=299), "row stride"), ("kcg_matmul_fp8", dict(b_scale_stride_row=-1), "negative"),
    ("kcg_matmul_fp8", dict(a_stride=(1 << 22) + 16), "apart"), ("kcg_matmul_fp8", dict(a_scale_stride_row=(1 << 20) + 1), "apart"),
    ("kcg_moe_layer", dict(tokens=65), "few tokens"), ("kcg_moe_layer", dict(tokens=-1), "tokens"), ("kcg_moe_layer", dict(experts=513), "experts"),
    ("kcg_moe_layer", dict(experts=0), "experts"), ("kcg_moe_layer", dict(topk=9), "topk"), ("kcg_moe_layer", dict(topk=17, experts=64), "topk"), ("kcg_moe_layer", dict(topk=0), "topk"),
    ("kcg_moe_layer", dict(hidden=72), "multiples of 16"), ("kcg_moe_layer", dict(inter=40), "multiples of 16"), ("kcg_moe_layer", dict(inter=0), "multiples of 16"),
    ("kcg_moe_layer", dict(dtype=F32), "e4m3"), ("kcg_moe_layer", dict(weight_dtype=BF16, dtype=F16), "both in bfloat16"), ("kcg_moe_layer", dict(weight_dtype=F16), "e4m3"),
    ("kcg_moe_layer", dict(x=0), "null"), ("kcg_moe_layer", dict(ids=0), "null"), ("kcg_moe_layer", dict(workspace=0), "null"), ("kcg_moe_layer", dict(w2_scale=0), "scales"),
    ("kcg_moe_layer", dict(workspace_bytes=100), "workspace"), ("kcg_moe_layer", dict(x=P + 1), "aligned"), ("kcg_moe_layer", dict(w13=P + 8), "16 bytes"),
    ("kcg_moe_layer", dict(w2_stride_row=56), "16 bytes"), ("kcg_moe_layer", dict(workspace=P + 4), "16 bytes"), ("kcg_moe_layer", dict(out_stride=32), "stride"),
    ("kcg_moe_layer", dict(w13_stride_expert=-16), "stride"),
]


def call(name, values):
    order = [n for n, _ in fields(name)]
    assert sorted(order) == sorted(values)
    _native.check(getattr(_native_ops.lib(), name)(STRUCTS[name].pack(*[values[n] for n in order]), 0, 0))


@pytest.mark.parametrize("name,change,text", BAD, ids=[f"{n[4:]}-{'-'.join(c)}-{i}" for i, (n, c, _) in enumerate(BAD)])
def test_refused_before_anything_is_launched(name, change, text):
    with pytest.raises(_native.KcgError, match=text) as e:
        call(name, {**GOOD[name], **change})
    assert e.value.status == _native.ERR_ARGUMENT


@pytest.mark.skipif(torch.cuda.is_available(), reason="says what happens without a GPU")
@pytest.mark.parametrize("name", list(STRUCTS))
def test_without_a_gpu_a_good_call_fails_loudly(name):
    with pytest.raises(_native.KcgError) as e:
        call(name, GOOD[name])
    assert e.value.status == _native.ERR_HIP
    with pytest.raises(_native.KcgError):
        _native_ops.load(0)


@pytest.mark.parametrize("name,change", [("kcg_rmsnorm_quant", dict(rows=0, x=0)), ("kcg_rmsnorm_quant", dict(cols=0)), ("kcg_swiglu_quant", dict(rows=0, q=0)),
                                         ("kcg_matmul_fp8", dict(m=0, a=0)), ("kcg_matmul_fp8", dict(n=0, c=0)), ("kcg_moe_layer", dict(tokens=0, x=0))])
def test_empty_calls_do_nothing(name, change):
    call(name, {**GOOD[name], **change})


@pytest.mark.parametrize("name", list(STRUCTS))
def test_null_arguments(name):
    assert getattr(_native_ops.lib(), name)(None, 0, 0) == _native.ERR_ARGUMENT


def test_workspace_of_the_experts():
    assert _native_ops.moe_workspace_bytes(0, 8, 2, 64, 48) == 0
    small, large = _native_ops.moe_workspace_bytes(1, 8, 2, 64, 48), _native_ops.moe_workspace_bytes(64, 8, 2, 64, 48)
    assert 0 < small < large and small % 16 == large % 16 == 0
    with pytest.raises(_native.KcgError):
        _native_ops.moe_workspace_bytes(65, 8, 2, 64, 48)


def test_no_cpu_path():
    q = torch.zeros(2, 128).to(torch.float8_e4m3fn)
    s = torch.ones(2, 1)
    with pytest.raises(TypeError, match="GPU"):
        rmsnorm_quant(torch.zeros(2, 128), torch.ones(128))
    with pytest.raises(TypeError, match="GPU"):
        swiglu_quant(torch.zeros(2, 256))
    with pytest.raises(TypeError, match="GPU"):
        matmul_fp8(q, s, q, s[:1])
    with pytest.raises(TypeError, match="GPU"):
        moe_layer(torch.zeros(1, 16), torch.zeros(1, 2), 1, torch.zeros(2, 32, 16), torch.zeros(2, 16, 16))


def test_the_tested_products_reach_every_kernel():
    """The sizes of tests/test_gpu_ops.py, by the kernel they run."""
    from tests.test_gpu_ops import KERNEL_SIZES, MATMULS
    reached = {_native_ops.matmul_fp8_kernel(m, n, k, c) for m, n, k in KERNEL_SIZES for c in (BF16, F16, F32)}
    with open(os.path.join(ROOT, "codegendemo_amd", "csrc", "kcg_ops.hsaco"), "rb") as f:
        built = {m.decode() for m in re.findall(rb"kcg_mm8_[a-z]+_[a-z0-9]+_[0-9x_]+(?=\0)", f.read())}
    assert len(built) == 3 * 10 + 6 and reached == built
    assert _native_ops.matmul_fp8_kernel(0, 5, 5, BF16) == ""
    assert all(_native_ops.matmul_fp8_kernel(m, n, k, BF16) for m, n, k, _ in MATMULS)
    with pytest.raises(_native.KcgError):
        _native_ops.matmul_fp8_kernel(1, 1, 1, F64)


@pytest.mark.parametrize("argv", [["--operator", "matmul_fp8", "--sizes", "1", "2"], ["--operator", "swiglu_quant", "--sizes", "0", "4"], ["--sizes", "4"], ["--operator", "softmax"]])
def test_operator_check_command_refuses(argv, capsys):
    from codegendemo_amd.kcg import test as single
    with pytest.raises(SystemExit) as e:
        single.main(argv)
    assert e.value.code == 2 and "error" in capsys.readouterr().err


@pytest.mark.parametrize("call", [
    lambda x: rmsnorm_quant(torch.zeros(2, 128), x[0]), lambda x: rmsnorm_quant(torch.zeros(2, 128), torch.zeros(128), residual=x), lambda x: swiglu_quant(x),
    lambda x: matmul_fp8(torch.zeros(2, 128), x, torch.zeros(2, 128), torch.zeros(1, 1)), lambda x: matmul_fp8(x.detach(), x.detach(), x.detach(), x.detach(), out=x),
    lambda x: moe_layer(torch.zeros(2, 16), x, 1, torch.zeros(128, 32, 16), torch.zeros(128, 16, 16)),
    lambda x: moe_layer(torch.zeros(2, 16), torch.zeros(2, 1), 1, x[None], torch.zeros(1, 16, 16))])
def test_a_tensor_that_requires_a_gradient_is_refused(call):
    """... before anything else; without gradients the same call gets as far as finding no GPU."""
    x = torch.zeros(2, 128, requires_grad=True)
    with pytest.raises(RuntimeError, match="no gradient.*no_grad"):
        call(x)
    with torch.no_grad(), pytest.raises(TypeError, match="GPU"):
        call(x)
    with torch.inference_mode(), pytest.raises(TypeError, match="GPU"):
        call(x)


def built_kernels(pattern):
    with open(os.path.join(ROOT, "codegendemo_amd", "csrc", "kcg_ops.hsaco"), "rb") as f:
        return {m.decode() for m in re.findall(rb"(?:%s)(?=\0)" % pattern, f.read())}


def parameters(test):
    """What a test is parametrised over: {names: values}."""
    return {m.args[0]: m.args[1] for m in test.pytestmark if m.name == "parametrize"}


def test_every_product_kernel_is_run():
    """From the very lists that the GPU tests run over, types included."""
    from tests import test_gpu_ops, test_gpu_ops_kernels
    codes = {torch.bfloat16: BF16, torch.float16: F16, torch.float32: F32}
    run = set()
    for test in (test_gpu_ops.test_matmul_kernels, test_gpu_ops_kernels.test_matmul_kernels_in_float16):
        p = parameters(test)
        run |= {_native_ops.matmul_fp8_kernel(m, n, k, codes[out]) for m, n, k in p["m,n,k"] for out in p["out"]}
    built = built_kernels(rb"kcg_mm8_[a-z]+_[a-z0-9]+_[0-9x_]+")
    assert built and run == built, sorted(built - run)


def test_every_norm_kernel_is_run():
    """A kernel's name says how many threads a row gets and how many vectors of 8 each holds (0: any number)."""
    from tests import test_gpu_ops, test_gpu_ops_kernels
    names = {torch.bfloat16: "bf16", torch.float16: "f16", torch.float32: "f32"}
    built = built_kernels(rb"kcg_norm_[a-z0-9]+_[0-9]+_[0-9]+")
    holds = sorted({(int(nt) * int(v) * 8 or 1 << 62, f"{nt}_{v}") for nt, v in (b.split("_")[3:] for b in built)})
    run = set()
    for test in (test_gpu_ops.test_norm, test_gpu_ops_kernels.test_norm_kernels):
        for _, h, dtype in parameters(test)["t,h,dtype"]:
            run.add(f"kcg_norm_{names[dtype]}_" + next(name for most, name in holds if h <= most))
    assert len(built) == 21 and run == built, sorted(built - run)


def test_the_library_is_built_without_hipcc(tmp_path):
    """The tuned products' host side needs a C++ compiler alone; the operators say what is missing, and refuse bad arguments as ever."""
    out = tmp_path / "libkcg_gemm.so"
    made = subprocess.run(["make", "-C", _native.CSRC_DIR, f"OUT={out}", f"HIPCC={tmp_path}/hipcc", str(out)], capture_output=True, text=True)
    assert made.returncode == 0, made.stderr
    assert "without the kernels of the operators" in made.stderr
    code = f"""
import ctypes
L = ctypes.CDLL({str(out)!r})
L.kcg_last_error.restype = L.kcg_version.restype = ctypes.c_char_p
assert L.kcg_version()
assert L.kcg_ops_load(0) == {_native.ERR_COMPILE}
assert b"without hipcc" in L.kcg_last_error()
assert L.kcg_matmul_fp8(None, 0, 0) == {_native.ERR_ARGUMENT}
"""
    run = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True)
    assert run.returncode == 0, run.stderr


def accepted(name, change):
    """The arguments pass every check: what fails then is finding a GPU."""
    if torch.cuda.is_available():
        pytest.skip("the addresses are not a GPU's")
    with pytest.raises(_native.KcgError) as e:
        call(name, {**GOOD[name], **change})
    assert e.value.status == _native.ERR_HIP, str(e.value)


@pytest.mark.parametrize("name", ["kcg_rmsnorm_quant", "kcg_swiglu_quant"])
def test_scales_that_lie_between_others_do_not_overlap(name):
    """Three groups a row, every second of 5 neighbours: 0 2 4, 5 7 9, ...; transposed the same; one further apart or closer is refused."""
    three = dict(cols=300, q_stride=304, **({"x_stride": 300, "residual_stride": 300, "residual_out_stride": 300, "y_stride": 300} if "norm" in name else {"gate_up_stride": 600}))
    accepted(name, dict(three, scale_stride_row=5, scale_stride_group=2))
    accepted(name, dict(three, scale_stride_row=2, scale_stride_group=7))
    for row, group in ((4, 2), (2, 6)):
        with pytest.raises(_native.KcgError, match="overlap"):
            call(name, {**GOOD[name], **three, "scale_stride_row": row, "scale_stride_group": group})


def test_one_expert_has_no_stride_to_another():
    """A view of a lone expert's weights may name any stride for it."""
    accepted("kcg_moe_layer", dict(experts=1, topk=1, w13_stride_expert=1, w2_stride_expert=3))
    for change in (dict(w13_stride_expert=1), dict(w2_stride_expert=3)):
        with pytest.raises(_native.KcgError, match="16 bytes"):
            call("kcg_moe_layer", {**GOOD["kcg_moe_layer"], **change})
