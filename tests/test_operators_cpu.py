"""The feed-forward operators without a GPU: what they refuse, their sizes, and how they are found."""

import ctypes
import random
import subprocess
import sys
from pathlib import Path

import pytest
import torch

REPO = Path(__file__).resolve().parent.parent
NAMES = ["gated_add_rmsnorm_fp4quant", "moe_expert_ffn", "nvfp4_gemm_epilogue", "nvfp4_grouped_gemm", "nvfp4_quantize_grouped"]


@pytest.fixture(scope="module")
def lib():
    from tirx_kernels import _native

    return _native.lib()


def _error():
    from tirx_kernels import _native

    return _native.last_error()


# Addresses that no call gets as far as reading: every case below is refused on the host.
P, ODD = 1 << 20, (1 << 20) + 4


@pytest.mark.parametrize("args,message", [
    ((P, P, P, P, P, None, None, P, -1, 128, 256, 1, 0, None), "rows >= 0"),
    ((P, P, P, P, P, None, None, P, 4, 12, 256, 1, 0, None), "N % 8"),
    ((P, P, P, P, P, None, None, P, 4, 128, 96, 1, 0, None), "K % 64"),
    ((P, P, P, P, P, None, None, P, 4, 0, 256, 1, 0, None), "N % 8"),
    ((P, P, P, P, P, None, None, P, 4, 128, 256, 7, 0, None), "out_dtype"),
    ((P, P, P, P, P, None, None, P, 4, 128, 256, 1, 5, None), "activation"),
    ((P, P, P, P, P, None, None, P, 4, 128, 256, 1, -1, None), "activation"),
    ((None, P, P, P, P, None, None, P, 4, 128, 256, 1, 0, None), "null"),
    ((P, P, P, P, None, None, None, P, 4, 128, 256, 1, 0, None), "null"),
    ((P, P, P, P, P, None, None, None, 4, 128, 256, 1, 0, None), "null"),
    ((P, P, ODD, P, P, None, None, P, 4, 128, 256, 1, 0, None), "16-byte"),
    ((P, P, P, P, P, ODD, None, P, 4, 128, 256, 1, 0, None), "16-byte"),
    ((P, P, P, P, P, None, ODD, P, 4, 128, 256, 1, 0, None), "16-byte"),
    ((P, P, P, P, P, None, None, P, 2147483600, 128, 256, 1, 0, None), "below 2^31"),
])
def test_gemm_epilogue_refuses(lib, args, message):
    assert lib.b2_nvfp4_gemm_epilogue(*args) == 1 and message in _error()


@pytest.mark.parametrize("args,message", [
    ((P, P, P, P, P, P, None, P, 4, 0, 128, 256, 1, 0, None), "1 to 384 groups"),
    ((P, P, P, P, P, P, None, P, 4, 385, 128, 256, 1, 0, None), "1 to 384 groups"),
    ((P, P, P, P, P, P, None, P, 4, 384, 1 << 23, 256, 1, 0, None), "below 2^31"),
    ((P, P, P, P, P, None, None, P, 4, 2, 128, 256, 1, 0, None), "null"),
    ((P, P, P, P, P, P, None, P, -4, 2, 128, 256, 1, 0, None), "rows >= 0"),
    ((P, P, P, P, P, P + 2, None, P, 4, 2, 128, 256, 1, 0, None), "4-byte"),
])
def test_grouped_gemm_refuses(lib, args, message):
    assert lib.b2_nvfp4_grouped_gemm(*args) == 1 and message in _error()


@pytest.mark.parametrize("args,message", [
    ((P, P, P, P, P, P, P, P, P, 4, 2, 64, 256, 1, None), "multiple of 128"),
    ((P, P, P, P, P, P, P, P, P, 4, 2, 0, 256, 1, None), "multiple of 128"),
    ((P, P, P, P, P, P, P, None, P, 4, 2, 128, 256, 1, None), "null"),
    ((P, P, P, P, P, P, None, P, P, 4, 2, 128, 256, 1, None), "null"),
    ((P, P, P, P, P, P, P, P, ODD, 4, 2, 128, 256, 1, None), "misaligned"),
    ((P, P, P, P, P, P, P, P, P, 4, 2, 128, 256, 3, None), "out_dtype"),
])
def test_gated_product_refuses(lib, args, message):
    assert lib.b2_nvfp4_grouped_gemm_gated(*args) == 1 and message in _error()


@pytest.mark.parametrize("args,message", [
    ((P, None, P, P, P, P, 4, 4, 2, 96, 1, 0, None), "k % 64"),
    ((P, None, P, P, P, P, 4, 4, 0, 128, 1, 0, None), "1 to 384 groups"),
    ((P, None, P, P, P, P, 3, 4, 2, 128, 1, 0, None), "without an index"),
    ((P, P, P, P, P, P, 4, 4, 2, 128, 9, 0, None), "in_dtype"),
    ((P, P, None, P, P, P, 4, 4, 2, 128, 1, 0, None), "null"),
    ((P + 8, P, P, P, P, P, 4, 4, 2, 128, 1, 0, None), "16-byte"),
    ((P, P, P, P, P, P, 4, 2147483600, 2, 128, 1, 0, None), "rows >= 0"),
])
def test_quantize_grouped_refuses(lib, args, message):
    assert lib.b2_nvfp4_quantize_grouped(*args) == 1 and message in _error()


def test_routing_entry_points_refuse(lib):
    assert lib.b2_moe_plan(P, P, P, P, 4, 0, 8, None) == 1 and "topk" in _error()
    assert lib.b2_moe_plan(P, P, P, P, 4, 2, 385, None) == 1 and "384" in _error()
    assert lib.b2_moe_plan(P, P, P, P, 1 << 30, 2, 8, None) == 1 and "2^31" in _error()
    assert lib.b2_moe_plan(P, None, P, P, 4, 2, 8, None) == 1 and "null" in _error()
    assert lib.b2_moe_plan(P + 1, P, P, P, 4, 2, 8, None) == 1 and "4-byte" in _error()
    assert lib.b2_moe_dispatch(P, P, P, P, P, P, P, P, 4, 33, 8, 128, 1, None) == 1 and "topk <= 32" in _error()
    assert lib.b2_moe_dispatch(P, P, P, P, P, P, P, P, 4, 2, 8, 96, 1, None) == 1 and "k % 64" in _error()
    assert lib.b2_moe_dispatch(P, P, P, P, None, P, P, P, 400, 2, 8, 128, 1, None) == 1 and "null" in _error()
    assert lib.b2_moe_dispatch(P, P, P, P, P, P, P, P, 4, 2, 8, 128, 4, None) == 1 and "dtype" in _error()
    assert lib.b2_moe_combine(P, P, P, None, P, 8, 4, 2, 12, 1, None) == 1 and "n % 8" in _error()
    assert lib.b2_moe_combine(P, P, P, None, P, 8, 4, 0, 16, 1, None) == 1 and "topk" in _error()
    assert lib.b2_moe_combine(None, P, P, None, P, 8, 4, 2, 16, 1, None) == 1 and "null" in _error()
    assert lib.b2_moe_combine(P, P, P, ODD, P, 8, 4, 2, 16, 1, None) == 1 and "16-byte" in _error()
    ffn = lambda **kw: lib.b2_moe_expert_ffn(*[kw.get(f"p{i}", P) for i in range(13)], kw.get("ws", P), kw.get("bytes", 1 << 40),
                                             *kw.get("sizes", (4, 2, 8, 128, 128)), kw.get("dtype", 1), None)
    assert ffn(sizes=(4, 2, 8, 96, 128)) == 1 and "hidden % 64" in _error()
    assert ffn(sizes=(4, 40, 8, 128, 128)) == 1 and "topk <= 32" in _error()
    assert ffn(dtype=2) == 1 and "dtype" in _error()
    assert ffn(bytes=100) == 1 and "workspace of" in _error()
    assert ffn(ws=P + 16) == 1 and "aligned to 256" in _error()
    assert ffn(ws=None) == 1 and "0 given" in _error()
    assert ffn(p3=None) == 1 and "null" in _error()
    assert ffn(p11=ODD) == 1 and "16-byte" in _error()


@pytest.mark.parametrize("args,message", [
    ((P, P, P, P, P, P, P, P, P, 4, 24, 1, 1.0, 1e-6, 1, 0, 0, None), "H % 16"),
    ((P, P, P, P, P, P, P, P, P, 4, 32784, 1, 1.0, 1e-6, 1, 0, 0, None), "H <= 32768"),
    ((P, P, P, P, P, P, P, P, P, -1, 64, 1, 1.0, 1e-6, 1, 0, 0, None), "M >= 0"),
    ((P, P, P, P, P, P, P, P, P, 4, 64, 0, 1.0, 1e-6, 1, 0, 0, None), "rows_per_gate >= 1"),
    ((P, P, P, P, P, P, P, P, P, 4, 64, 1, 1.0, 1e-6, 2, 0, 0, None), "in_dtype"),
    ((P, P, P, P, P, P, P, None, None, 4, 64, 1, 1.0, 1e-6, 1, 1, 0, None), "null"),
    ((P, P, P, P, None, P, P, P, P, 4, 64, 1, 1.0, 1e-6, 1, 0, 0, None), "null"),
    ((P + 16, P, P, P, P, P, P, P, P, 4, 64, 1, 1.0, 1e-6, 1, 0, 0, None), "32-byte"),
    ((P, P, P, P, P, P, P + 16, P, P, 4, 64, 1, 1.0, 1e-6, 1, 0, 0, None), "32-byte"),
])
def test_gated_norm_refuses(lib, args, message):
    assert lib.b2_gated_add_rmsnorm_fp4quant(*args) == 1 and message in _error()


def test_nothing_to_do_is_no_error(lib):
    assert lib.b2_nvfp4_gemm_epilogue(None, None, None, None, None, None, None, None, 0, 128, 256, 1, 0, None) == 0
    assert lib.b2_nvfp4_grouped_gemm(None, None, None, None, None, None, None, None, 0, 4, 128, 256, 1, 0, None) == 0
    assert lib.b2_nvfp4_quantize_grouped(None, None, None, None, None, None, 0, 0, 4, 128, 1, 0, None) == 0
    assert lib.b2_moe_dispatch(None, None, None, None, None, None, None, None, 0, 2, 8, 128, 1, None) == 0
    assert lib.b2_moe_combine(None, None, None, None, None, 0, 0, 2, 16, 1, None) == 0
    assert lib.b2_gated_add_rmsnorm_fp4quant(*[None] * 9, 0, 64, 1, 1.0, 1e-6, 1, 0, 0, None) == 0


def test_size_helpers(lib):
    from tirx_kernels import _checks
    from tirx_kernels.basic import moe_ffn

    for rows, groups, k in [(0, 1, 64), (1, 64, 4096), (777, 7, 1088), (16384, 384, 2048)]:
        assert lib.b2_nvfp4_grouped_sf_bytes(rows, groups, k) == _checks.grouped_sf_numel(rows, groups, k)
    assert lib.b2_nvfp4_grouped_sf_bytes(4, 0, 64) == -1 and lib.b2_nvfp4_grouped_sf_bytes(4, 2, 96) == -1
    assert moe_ffn.workspace_bytes(0, 2, 8, 128, 128) > 0
    fused, apart = moe_ffn.workspace_bytes(1000, 2, 8, 512, 256), moe_ffn.workspace_bytes(1000, 2, 8, 512, 320)
    assert apart - fused > 2000 * 320 * 4  # only there the 16-bit product lies in memory
    with pytest.raises(ValueError):
        moe_ffn.workspace_bytes(4, 2, 8, 100, 128)


def test_group_tiles_never_meet():
    """A group begins at tile offset // 128 + group: behind the last tile of the group in front, and inside the buffer."""
    rng = random.Random(0)
    for _ in range(300):
        groups = rng.choice([1, 2, 7, 64, 384])
        sizes = [rng.choice([0, 0, 1, 5, 127, 128, 129, 255, 256, rng.randrange(2000)]) for _ in range(groups)]
        offset, end = 0, 0
        for g, size in enumerate(sizes):
            first = offset // 128 + g
            assert first >= end
            end = first + -(-size // 128) if size else end
            offset += size
        assert end <= offset // 128 + groups


def _tensors(**shapes):
    return {k: torch.zeros(s, dtype=d) for k, (s, d) in shapes.items()}


def test_modules_refuse_configurations():
    from tirx_kernels import registry

    load = lambda name: registry.load_kernel(name, strict=True)
    bad = {
        "nvfp4_gemm_epilogue": [dict(M=-1, N=8, K=64), dict(M=1, N=12, K=64), dict(M=1, N=8, K=96), dict(M=1, N=8, K=64, activation="tanh"),
                                dict(M=1, N=8, K=64, out_dtype="float32")],
        "nvfp4_grouped_gemm": [dict(rows=1, groups=0, N=8, K=64), dict(rows=1, groups=385, N=8, K=64), dict(rows=-1, groups=1, N=8, K=64),
                               dict(rows=1, groups=1, N=4, K=64), dict(rows=1, groups=1, N=8, K=64, out_dtype="float32")],
        "nvfp4_quantize_grouped": [dict(dtype="float32", in_rows=1, rows=1, groups=1, k=64), dict(dtype="float16", in_rows=1, rows=1, groups=1, k=32),
                                   dict(dtype="float16", in_rows=1, rows=1, groups=500, k=64), dict(dtype="float16", in_rows=-1, rows=1, groups=1, k=64)],
        "moe_expert_ffn": [dict(tokens=1, topk=0, experts=4, hidden=64, inner=64), dict(tokens=1, topk=1, experts=4, hidden=96, inner=64),
                           dict(tokens=1, topk=1, experts=400, hidden=64, inner=64), dict(tokens=1, topk=1, experts=4, hidden=64, inner=64, dtype="float32")],
        "gated_add_rmsnorm_fp4quant": [dict(input_dtype="float32", M=1, H=64), dict(input_dtype="float16", M=1, H=24), dict(input_dtype="float16", M=1, H=40000),
                                       dict(input_dtype="float16", M=1, H=64, rows_per_gate=0)],
    }
    for name, configs in bad.items():
        for config in configs:
            with pytest.raises(ValueError):
                load(name).get_kernel(**config)


def test_executables_refuse_tensors():
    from tirx_kernels import registry

    ex = registry.load_kernel("nvfp4_gemm_epilogue").get_kernel(M=4, N=8, K=64).config["launcher"]
    u8, f32, bf16 = torch.uint8, torch.float32, torch.bfloat16
    t = _tensors(A=((4, 32), u8), B=((8, 32), u8), SFA=((512,), u8), SFB=((512,), u8), alpha=((1,), f32), D=((4, 8), bf16))
    call = lambda **kw: ex(*[{**t, "bias": None, "residual": None, **kw}[k] for k in ("A", "B", "SFA", "SFB", "alpha", "bias", "residual", "D")])
    for change, message in [({}, "A: all tensors must be CUDA"), ({"A": torch.zeros(4, 16, dtype=u8)}, r"A must have shape \(4, 32\)"),
                            ({"A": None}, "A must be a tensor"), ({"A": t["A"].float()}, "A must be torch.uint8")]:
        with pytest.raises(ValueError, match=message):
            call(**change)
    from tirx_kernels import _checks

    for spec, tensor, message in [(ex.specs[2], torch.zeros(100, dtype=u8), "SFA must have 512 elements"), (ex.specs[4], 1.0, "alpha must be a tensor"),
                                  (ex.specs[5], torch.zeros(8), "bias must be torch.bfloat16"), (ex.specs[7], None, "D must be a tensor")]:
        with pytest.raises(ValueError, match=message):
            _checks.require_tensors((spec,), (tensor,))
    ex = registry.load_kernel("gated_add_rmsnorm_fp4quant").get_kernel("float16", 2, 64, quantize=False).config["launcher"]
    x = torch.zeros(2, 64, dtype=torch.float16)
    with pytest.raises(ValueError, match="quantized form"):
        ex(x, x, None, None, x[0], x, x, x, None, 1.0, 1e-6)
    from tirx_kernels.basic import moe_ffn

    ids = torch.zeros(3, 2, dtype=torch.int32)
    for refused in (lambda: moe_ffn.plan(ids, 0), lambda: moe_ffn.plan(ids[0], 4), lambda: moe_ffn.plan(ids.long(), 4), lambda: moe_ffn.plan(ids, 4),
                    lambda: moe_ffn.combine(torch.zeros(6, 12), ids, torch.zeros(3, 2)), lambda: moe_ffn.combine(torch.zeros(6, 12, dtype=bf16), ids, torch.zeros(3, 2)),
                    lambda: moe_ffn.dispatch(torch.zeros(3, 64, dtype=bf16), ids, torch.ones(4)),
                    lambda: moe_ffn.dispatch(torch.zeros(3, 64, dtype=bf16), torch.zeros(3, 33, dtype=torch.int32), torch.ones(4)),
                    lambda: moe_ffn.gated_product(torch.zeros(6, 32, dtype=u8), None, None, torch.zeros(4, 64, 32, dtype=u8), None, None, None)):
        with pytest.raises(ValueError):
            refused()
    with pytest.raises(ValueError, match="CUDA"):
        moe_ffn.ExpertWeights(torch.zeros(2, 256, 64, dtype=u8), torch.zeros(2 * 256 * 8, dtype=u8), torch.zeros(2), torch.zeros(2),
                              torch.zeros(2, 128, 64, dtype=u8), torch.zeros(2 * 128 * 8, dtype=u8), torch.zeros(2), torch.zeros(2))
    with pytest.raises(ValueError, match="w2 must have shape"):
        _checks.require_tensors(moe_ffn._weight_specs(2, 128, 128)[4:5], (torch.zeros(2, 64, 64, dtype=u8),))
    with pytest.raises(ValueError, match="must be"):
        moe_ffn.ExpertWeights(torch.zeros(2, 256, dtype=u8), None, None, None, torch.zeros(2, 128, 64, dtype=u8), None, None, None)


def test_operators_are_found_by_name_beside_the_registry():
    from tirx_kernels import registry

    index = registry.operator_index(strict=True)
    assert sorted(index) == NAMES and not set(index) & set(registry.kernel_index(strict=True))
    for name in NAMES:
        module = registry.load_kernel(name, strict=True)
        assert registry.module_meta(module)["name"] == name
        for configs in (module.CONFIGS, module.BENCH_CONFIGS):
            labels = [c["label"] for c in configs]
            assert len(labels) == len(set(labels))
            for config in configs:
                assert module.get_kernel(**{k: v for k, v in config.items() if k != "label"}).symbol.startswith("b2_")


def test_command_lines_take_operator_names():
    env = {"PYTHONPATH": f"{REPO / 'tirx-kernels_b200'}:{REPO}", "PATH": "/usr/bin:/bin"}
    run = lambda *a: subprocess.run([sys.executable, "-m", *a], capture_output=True, text=True, env=env)
    nothing = run("tirx_kernels.test", "--kernel", "nvfp4_grouped_gemm", "--config", "no_such_label", "--json")
    assert nothing.returncode == 2 and "no kernel configs matched" in nothing.stdout
    other = run("tirx_kernels.test", "--kernel", "nvfp4_grouped_gemm", "--cc", "9")
    assert other.returncode == 1 and "not found" in other.stdout


def test_set_variant_refuses(lib):
    assert lib.b2_nvfp4_grouped_gemm_set_variant(6) == 1 and "variant 6" in _error()
    assert lib.b2_nvfp4_grouped_gemm_set_variant(-2) == 1
    assert lib.b2_nvfp4_grouped_gemm_set_variant(-1) == 0


def test_every_operator_argument_list_matches_the_header():
    """ctypes knows as many arguments as the header declares."""
    import re

    from tirx_kernels import _native

    header = re.sub(r"/\*.*?\*/", "", (REPO / "include" / "b200_nvfp4.h").read_text(), flags=re.S)
    for name in _native.MAIN_SIGNATURES:
        declared = re.search(rf"\b{name}\s*\(([^;]*)\)\s*;", header).group(1)
        count = 0 if declared.strip() in ("", "void") else declared.count(",") + 1
        assert count == len(_native.MAIN_SIGNATURES[name][1]), name
    assert ctypes.sizeof(ctypes.c_void_p) == 8


def test_bound_calls_refuse_what_they_are_not_made_for():
    """The compiled half of a call: counts and kinds when it is bound, tensors and counts when it is called; nothing is launched."""
    from tirx_kernels import _checks, _native

    bind = _native._binding().bind
    spec = _checks.tensor_spec
    specs = tuple(spec(n, "uint8", -1) for n in ("A", "B", "SFA", "SFB")) + (spec("alpha", "float32", 1), spec("bias", "bfloat16", (8,), True),
                                                                              spec("residual", "bfloat16", (4, 8), True), spec("D", "bfloat16", (4, 8)))
    for symbol, address, some, sizes in [("b2_nvfp4_gemm", 1, specs, (1,) * 5), ("b2_nvfp4_gemm_epilogue", 0, specs, (1,) * 5),
                                         ("b2_nvfp4_gemm_epilogue", 1, specs[:7], (1,) * 5), ("b2_nvfp4_gemm_epilogue", 1, specs, (1,) * 4),
                                         ("b2_nvfp4_gemm_epilogue", 1, specs, (1, 1, 1, 1, 0.5)), (None, 0, specs, (1,)), (None, 0, specs * 3, ()),
                                         (None, 0, (("A", "uint8", 1, False),), ()), (None, 0, (("A", torch.uint8, "x", False),), ()),
                                         (None, 0, [], ())]:
        with pytest.raises(TypeError):
            bind(symbol, address, some, sizes)
    check = bind(None, 0, (spec("a", "float32", (2, 3)), spec("b", "int32", 4, True)), ())
    a = torch.zeros(2, 3)
    for tensors in [(a, None), (None, None), (1, None), ("a", None), (a.double(), None), (torch.empty(2, 3, device="meta"), None),
                    (a, torch.zeros(4, dtype=torch.int32))]:
        assert check(*tensors) == -1
    assert bind(None, 0, (spec("b", "int32", 4, True),), ())(None) == 0
    for arguments in [(), (a,), (a, None, None)]:
        with pytest.raises(TypeError):
            check(*arguments)
    with pytest.raises(TypeError):
        check(a, b=None)
    with pytest.raises(ValueError, match="a: all tensors must be CUDA"):
        _native.Launch(None, (spec("a", "float32", (2, 3)),))(a)


@pytest.mark.parametrize("stages,issuers,safe", [(3, 1, True), (4, 1, True), (2, 2, True), (4, 2, True), (6, 2, True), (3, 2, False), (5, 2, False)])
def test_ring_of_two_issuers_is_even(stages, issuers, safe):
    """All orders in which slabs land and are consumed: a wait by phase parity never passes for a slab that has not landed.

    Slab n lies in stage n % stages, its load is issued when the slab before it in that stage was consumed, loads land in any
    order, issuer n % issuers consumes slab n when the parity test of the stage's barrier passes: phases completed there and
    the phase asked for, n // stages, differ in parity, or (the stale case) the test sees the phase in front of an open one."""
    slabs = 3 * stages
    seen, todo = set(), [(0, tuple(range(issuers)))]  # bit mask of landed slabs, next slab of every issuer
    stale = False
    while todo and not stale:
        state = todo.pop()
        if state in seen:
            continue
        seen.add(state)
        landed, heads = state
        consumed = lambda n: n < heads[n % issuers]
        issued = 0
        while issued < slabs and (issued < stages or consumed(issued - stages)):
            issued += 1  # in order
        for n in range(issued):
            if not landed >> n & 1:
                todo.append((landed | 1 << n, heads))
        for i, n in enumerate(heads):
            if n >= slabs:
                continue
            completed = sum(landed >> m & 1 for m in range(n % stages, slabs, stages))  # phases of the stage's barrier
            if completed % 2 != n // stages % 2:
                stale = stale or not landed >> n & 1
                todo.append((landed, heads[:i] + (n + issuers,) + heads[i + 1:]))
    assert stale != safe
