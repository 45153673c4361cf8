"""GPU parity of the feed-forward operators: every module's own configurations against its 64-bit formula."""

import dataclasses

import pytest

pytestmark = pytest.mark.gpu

OPERATORS = ["gated_add_rmsnorm_fp4quant", "nvfp4_quantize_grouped", "nvfp4_gemm_epilogue", "nvfp4_grouped_gemm", "moe_expert_ffn"]


def _cases():
    from tirx_kernels import registry

    return [pytest.param(name, config, id=f"{name}-{config['label']}") for name in OPERATORS
            for config in registry.load_kernel(name).CONFIGS]


@pytest.mark.parametrize("name,config", _cases())
def test_configs_pass_run_test(name, config, native):
    from tirx_kernels import registry
    from tirx_kernels.runner import run_kernel_test

    run_kernel_test(name, config, registry={name: registry.load_kernel(name)})


import torch  # noqa: E402


@pytest.fixture()
def variant(native):
    yield native.nvfp4_grouped_gemm_set_variant
    native.nvfp4_grouped_gemm_set_variant(-1)


def _launcher(module, **config):
    from tirx_kernels.runner import compile_kernel

    return compile_kernel(module.get_kernel(**config))


# ---- product with its epilogue --------------------------------------------------------------------------------------


def _linear(M, N, K, activation="none", out_dtype="bfloat16", bias=True, residual=True, in_place=False, data=None):
    """(output, float64 formula, tolerance)."""
    from tirx_kernels import _native
    from tirx_kernels.basic import nvfp4_gemm_epilogue as mod

    data = data or mod.prepare_data(M, N, K, out_dtype=out_dtype, bias=bias, residual=residual)
    want, size = mod.expected(*data, activation)
    D = data[6] if in_place else torch.full((M, N), float("nan"), dtype=getattr(torch, out_dtype), device="cuda")
    _launcher(mod, M=M, N=N, K=K, activation=activation, out_dtype=out_dtype)(*data, D)
    torch.cuda.synchronize()
    _native.nvfp4_grouped_gemm_status()
    return D, want, mod.tolerance(want, size, K, out_dtype)


def _near(got, want, tolerance):
    excess = ((got.double() - want).abs() - tolerance).max().item()
    assert excess <= 0, f"off by {excess:.3e} more than the tolerance"


# one row and column block; rows and columns that end inside tiles of every size; K of part of a slab, of a slab, beyond the ring
SHAPES = [(1, 8, 64), (33, 72, 320), (129, 136, 192), (257, 264, 576), (300, 1000, 256), (31, 520, 3136), (200, 640, 64)]


@pytest.mark.parametrize("which", [0, 1, 2, 3, 4, 5])
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_linear_every_variant(which, M, N, K, variant):
    variant(which)
    _near(*_linear(M, N, K, "none", ["bfloat16", "float16"][which % 2]))


@pytest.mark.parametrize("which", [-1, 0, 2, 4, 5])
@pytest.mark.parametrize("activation", ["none", "relu", "gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("bias,residual", [(False, False), (True, False), (False, True)])
def test_linear_epilogues(which, activation, bias, residual, variant):
    variant(which)
    _near(*_linear(150, 200, 448, activation, "float16" if bias else "bfloat16", bias, residual))


@pytest.mark.parametrize("which", [0, 1, 2, 3, 4, 5])
def test_linear_residual_may_be_the_output(which, variant):
    variant(which)
    _near(*_linear(260, 328, 512, "silu", in_place=True))


def test_linear_many_tiles_per_cta(variant):
    """More tiles than SMs: accumulators, barriers and staging are used again and again, residual and bias with them."""
    for which in (1, 3, 4, 5):
        variant(which)
        _near(*_linear(1100, 6000, 192, "gelu_tanh"))


def test_linear_ignores_what_lies_in_padding():
    """Scale bytes of rows that do not exist may be NaN: the same output."""
    from tirx_kernels.basic import nvfp4_gemm_epilogue as mod

    for M, N in ((5, 72), (150, 200), (300, 520)):
        data = mod.prepare_data(M, N, 320)
        clean, want, tolerance = _linear(M, N, 320, data=data)
        from tirx_kernels import _checks

        for sf, rows in ((data[2], M), (data[3], N)):
            sf[_checks.padding_mask(rows, 320 // 16, "128x4", sf.device)] = 0x7F
        dirty, _, _ = _linear(M, N, 320, data=data)
        _near(clean, want, tolerance)
        assert torch.equal(clean, dirty)


def test_linear_nan_and_infinity_stay_where_they_are():
    from tirx_kernels.basic import nvfp4_gemm_epilogue as mod

    data = list(mod.prepare_data(70, 136, 256))
    clean, _, _ = _linear(70, 136, 256, "relu", data=data)
    data[5], data[6] = data[5].clone(), data[6].clone()
    data[5][9], data[5][11], data[5][13] = float("nan"), float("inf"), float("-inf")
    data[6][40, 50], data[6][41, 51] = float("nan"), float("inf")
    D, _, _ = _linear(70, 136, 256, "relu", data=data)
    touched = torch.zeros(70, 136, dtype=torch.bool, device="cuda")
    touched[:, [9, 11, 13]] = True
    touched[40, 50] = touched[41, 51] = True
    assert torch.equal(D[~touched], clean[~touched])
    assert D[:, 9].isnan().all() and (D[:, 11] == float("inf")).all() and D[40, 50].isnan() and D[41, 51] == float("inf")
    assert torch.equal(D[:, 13], data[6][:, 13])  # relu(-inf) = 0


@pytest.mark.parametrize("activation,low,high", [("silu", 0.0, 1e4), ("gelu", 0.0, 1e4), ("gelu_tanh", 0.0, 1e4), ("relu", 0.0, 1e4)])
def test_linear_activations_far_out(activation, low, high):
    """Values of +-10000 from the bias: the activation's limits, no NaN from an exponential that overflows."""
    from tirx_kernels.basic import nvfp4_gemm_epilogue as mod

    data = list(mod.prepare_data(8, 16, 64, out_dtype="bfloat16", residual=False))
    data[4] = torch.zeros(1, device="cuda")
    data[5] = torch.tensor([-1e4, 1e4] * 8, device="cuda").bfloat16()
    D, _, _ = _linear(8, 16, 64, activation, data=data)
    assert (D[:, 0::2] == low).all() and torch.equal(D[:, 1::2], data[5][1::2].expand(8, 8))


def test_linear_zero_rows():
    from tirx_kernels.basic import nvfp4_gemm_epilogue as mod

    e = lambda *s, dtype=torch.uint8: torch.zeros(*s, dtype=dtype, device="cuda")
    ex = _launcher(mod, M=0, N=8, K=64)
    ex(e(0, 32), e(8, 32), e(0), e(512), e(1, dtype=torch.float32), None, None, e(0, 8, dtype=torch.bfloat16))
    torch.cuda.synchronize()


def test_linear_equals_the_plain_gemm_bit_for_bit(native):
    """Without bias, activation and residual the sums are those of nvfp4_gemm in tiles that add K in the same order."""
    from tirx_kernels.basic import nvfp4_gemm_epilogue as mod

    data = mod.prepare_data(2048, 2048, 1024, bias=False, residual=False)
    plain = torch.empty(2048, 2048, dtype=torch.bfloat16, device="cuda")
    native.nvfp4_gemm(*data[:5], plain, 2048, 2048, 1024)
    assert torch.equal(_linear(2048, 2048, 1024, data=data)[0], plain)


def test_linear_refuses_strides_and_other_places():
    from tirx_kernels.basic import nvfp4_gemm_epilogue as mod

    data = mod.prepare_data(32, 64, 128)
    D = torch.empty(32, 64, dtype=torch.bfloat16, device="cuda")
    ex = _launcher(mod, M=32, N=64, K=128)
    wide = torch.empty(32, 128, dtype=torch.bfloat16, device="cuda")[:, :64]
    with pytest.raises(ValueError, match="contiguous"):
        ex(*data, wide)
    with pytest.raises(ValueError, match="contiguous"):
        ex(*data[:6], data[6].t().contiguous().t(), D)
    with pytest.raises(ValueError, match="CUDA"):
        ex(*data, D.cpu())
    with pytest.raises(ValueError, match="16-byte"):
        shifted = torch.empty(32 * 64 + 4, dtype=torch.bfloat16, device="cuda")[4:].view(32, 64)
        ex(*data, shifted)
    with pytest.raises(ValueError, match="bias must be"):
        ex(*data[:5], data[5].half(), data[6], D)


# ---- grouped product ------------------------------------------------------------------------------------------------

SIZES = [[0, 0, 5, 0, 130, 1, 0], [257, 0, 31, 33, 128], [1] * 40, [0, 300], [64], [0, 0, 0], [129, 127, 255, 256, 3]]


@pytest.mark.parametrize("which", [-1, 1, 3, 4, 5])
@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: "-".join(map(str, s[:8])))
def test_grouped_every_variant(which, sizes, variant):
    from tirx_kernels.basic import nvfp4_grouped_gemm as mod

    variant(which)
    mod.run_test(max(1, sum(sizes)), len(sizes), 200, 448, ["gelu", "silu"][which % 2], ["bfloat16", "float16"][which % 2], True, sizes=sizes)


def test_grouped_many_groups_and_tiles(variant):
    from tirx_kernels.basic import nvfp4_grouped_gemm as mod

    for which in (1, 3, 4, 5):
        variant(which)
        mod.run_test(3000, 384, 264, 128, bias=False)
        mod.run_test(2000, 3, 4104, 64, bias=False)


@pytest.mark.parametrize("K", [960, 1024, 1088, 2048])
@pytest.mark.parametrize("activation,out_dtype", [("none", "bfloat16"), ("gelu", "float16")])
def test_grouped_few_rows_on_both_sides_of_the_split_epilogue(K, activation, out_dtype, variant):
    from tirx_kernels.basic import nvfp4_grouped_gemm as mod

    variant(1)
    mod.run_test(230, 12, 328, K, activation, out_dtype, True, sizes=[0, 1, 32, 33, 64, 7, 0, 31, 2, 60, 0, 0])
    mod.run_test(40, 40, 4096, K, bias=False, sizes=[1] * 40)


@pytest.mark.parametrize("which", [1, 3, 4])
def test_grouped_more_row_tiles_than_are_mapped(which, variant):
    """Behind the row tiles whose group is looked up (512 of single CTAs, 128 of pairs) it is searched."""
    from tirx_kernels.basic import nvfp4_grouped_gemm as mod

    variant(which)
    mod.run_test(70000 if which == 3 else 20000, 300, 136, 64, bias=False)
    sizes = [0] * 384
    sizes[0], sizes[200], sizes[383] = 40000, 1, 39000
    mod.run_test(79001, 384, 72, 64, bias=False, sizes=sizes)


def test_grouped_leaves_other_rows_alone():
    """Rows in front of offsets[0] and behind offsets[groups] keep their bytes, in every tile they share with a group."""
    from tirx_kernels import _checks, _native
    from tirx_kernels.basic import nvfp4_grouped_gemm as mod

    A, B, SFA, SFB, alpha, offsets, _ = mod.prepare_data(700, 3, 136, 256, bias=False, sizes=[100, 250, 50])
    moved = (offsets + 37).int()
    whole = torch.full((700, 136), 7.0, dtype=torch.bfloat16, device="cuda")
    rows = torch.cat([torch.arange(37, device="cuda"), torch.arange(437, 700, device="cuda")])
    A2 = torch.randint(0, 255, (700, 128), dtype=torch.uint8, device="cuda")
    A2[37:437] = A[:400]
    SFA2 = torch.full((_checks.grouped_sf_numel(700, 3, 256),), 0x7F, dtype=torch.uint8, device="cuda")
    old = _checks.logical_scale_bytes(SFA, SFA.numel() // 16, 16, "128x4")
    at = _checks.sf_offsets("128x4", SFA2.numel() // 16, 16, "cuda")
    g, frm = _checks.grouped_sf_rows(offsets, 400)
    to = (moved[:-1].long()[g] // 128 + g) * 128 + torch.arange(400, device="cuda") - offsets.long()[g]
    SFA2[at[to].reshape(-1)] = old[frm].reshape(-1)
    ref = torch.empty(700, 136, dtype=torch.bfloat16, device="cuda")
    ex = _launcher(mod, rows=700, groups=3, N=136, K=256)
    ex(A, B, SFA, SFB, alpha, offsets, None, ref)
    for which in (1, 3, 4, 5):
        _native.nvfp4_grouped_gemm_set_variant(which)
        whole.fill_(7.0)
        ex(A2, B, SFA2, SFB, alpha, moved, None, whole)
        torch.cuda.synchronize()
        assert (whole[rows] == 7.0).all() and torch.equal(whole[37:437], ref[:400])
    _native.nvfp4_grouped_gemm_set_variant(-1)


def test_grouped_offsets_out_of_range_are_clamped():
    """Offsets that fall or leave the rows are brought back by the kernel's own checks; what they do not cover stays."""
    from tirx_kernels import _native
    from tirx_kernels.basic import nvfp4_grouped_gemm as mod

    A, B, SFA, SFB, alpha, offsets, _ = mod.prepare_data(300, 3, 136, 256, bias=False, sizes=[100, 150, 50])
    D = torch.full((300, 136), 7.0, dtype=torch.bfloat16, device="cuda")
    ex = _launcher(mod, rows=300, groups=3, N=136, K=256)
    bad = torch.tensor([-5, 40, 20, 1 << 30], dtype=torch.int32, device="cuda")
    for which in (1, 3, 4, 5):
        _native.nvfp4_grouped_gemm_set_variant(which)
        ex(A, B, SFA, SFB, alpha, bad, None, D)
    bad = torch.tensor([250, 250, 10, 10], dtype=torch.int32, device="cuda")
    D.fill_(7.0)
    ex(A, B, SFA, SFB, alpha, bad, None, D)
    torch.cuda.synchronize()
    _native.nvfp4_grouped_gemm_set_variant(-1)
    _native.nvfp4_grouped_gemm_status()
    assert (D == 7.0).all()


def test_one_group_is_the_dense_product():
    from tirx_kernels.basic import nvfp4_gemm_epilogue as dense, nvfp4_grouped_gemm as mod

    A, B, SFA, SFB, alpha, bias, _ = dense.prepare_data(500, 392, 704, residual=False)
    want = _linear(500, 392, 704, "silu", data=[A, B, SFA, SFB, alpha, bias, None])[0]
    tiles = torch.zeros((500 // 128 + 1) * 128 * 44, dtype=torch.uint8, device="cuda")
    tiles[: SFA.numel()] = SFA
    D = torch.empty_like(want)
    offsets = torch.tensor([0, 500], dtype=torch.int32, device="cuda")
    _launcher(mod, rows=500, groups=1, N=392, K=704, activation="silu")(A, B[None], tiles, SFB, alpha, offsets, bias[None], D)
    assert torch.equal(D, want)


# ---- quantizer, plan, dispatch, gated product, weighted sum --------------------------------------------------------------


@pytest.mark.parametrize("dtype,silu", [("bfloat16", False), ("float16", False), ("bfloat16", True), ("float16", True)])
@pytest.mark.parametrize("rows,groups,k", [(1, 1, 64), (130, 5, 192), (300, 64, 2112), (40, 384, 8256)])
def test_quantize_grouped_shapes(dtype, silu, rows, groups, k):
    from tirx_kernels.basic import nvfp4_quantize_grouped as mod

    mod.run_test(dtype, max(1, rows // 2), rows, groups, k, silu)


def test_quantize_grouped_odd_indices_alignment_and_tail():
    from tirx_kernels import _checks
    from tirx_kernels.basic import nvfp4_quantize_grouped as mod

    k, rows, groups = 320, 12, 2
    x = torch.randn(6 * k + 8, device="cuda").bfloat16()[8:].view(6, k)  # 16-byte aligned, not 32
    index = torch.tensor([0, 0, 5, -1, 6, 1 << 30, 3, 3, 3, 1, 2, 4], dtype=torch.int32, device="cuda")
    offsets = torch.tensor([0, 4, 9], dtype=torch.int32, device="cuda")
    gs = torch.tensor([400.0, 500.0], device="cuda")
    out = torch.full((rows, k // 2), 0xA5, dtype=torch.uint8, device="cuda")
    sf = torch.full((_checks.grouped_sf_numel(rows, groups, k),), 0xA5, dtype=torch.uint8, device="cuda")
    _launcher(mod, dtype="bfloat16", in_rows=6, rows=rows, groups=groups, k=k)(x, index, offsets, out, sf, gs)
    assert torch.equal(out[0], out[1]) and torch.equal(out[6], out[7]) and not torch.equal(out[0], out[2])
    assert (out[[3, 4, 5]] == 0).all() and (out[9:] == 0xA5).all()
    tiles = _checks.logical_scale_bytes(sf, sf.numel() // (k // 16), k // 16, "128x4")
    assert (tiles[[3, 128, 129]] == 0).all() and (tiles[4:128] == 0xA5).all() and (tiles[133:] == 0xA5).all()
    assert (tiles[:3] != 0).all() and (tiles[130:133] != 0).all()


def _plan_want(ids, experts):
    flat = ids.flatten().cpu().long()
    valid = (flat >= 0) & (flat < experts)
    order = torch.sort(torch.where(valid, flat, experts), stable=True).indices[: int(valid.sum())]
    position = torch.full_like(flat, -1)
    position[order] = torch.arange(order.numel())
    row_token = torch.full_like(flat, -1)
    row_token[: order.numel()] = order // ids.shape[1]
    offsets = torch.zeros(experts + 1, dtype=torch.long)
    offsets[1:] = torch.bincount(flat[valid], minlength=experts).cumsum(0)
    return offsets, row_token, position.view(ids.shape)


PLANS = [(0, 2, 4), (1, 1, 1), (1, 8, 64), (7, 3, 5), (64, 8, 64), (65, 8, 384), (513, 1, 7), (1000, 4, 256), (5000, 6, 33)]


@pytest.mark.parametrize("tokens,topk,experts", PLANS)
def test_plan(tokens, topk, experts):
    from tirx_kernels.basic import moe_ffn

    g = torch.Generator().manual_seed(tokens + topk)
    for low, high in ((0, experts), (-2, experts + 3), (0, 1)):  # every id valid; some dropped; all the same
        ids = torch.randint(low, high, (tokens, topk), generator=g, dtype=torch.int32).cuda()
        got = moe_ffn.plan(ids, experts)
        for a, b in zip(got, _plan_want(ids, experts)):
            assert torch.equal(a.cpu().long(), b)
        again = moe_ffn.plan(ids, experts)
        assert all(torch.equal(a, b) for a, b in zip(got, again))


@pytest.mark.parametrize("tokens,topk,experts,hidden", [(1, 8, 64, 4096), (3, 2, 5, 64), (64, 8, 64, 320), (129, 4, 33, 2048), (700, 3, 384, 192), (3000, 2, 7, 128)])
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
def test_dispatch_is_plan_and_quantizer(tokens, topk, experts, hidden, dtype):
    from tirx_kernels import _checks
    from tirx_kernels.basic import moe_ffn, nvfp4_quantize_grouped as quantize

    g = torch.Generator().manual_seed(tokens)
    ids = torch.randint(-1, experts + 1, (tokens, topk), generator=g, dtype=torch.int32).cuda()
    x = torch.randn(tokens, hidden, generator=g).to(getattr(torch, dtype)).cuda()
    scales = 300 + 300 * torch.rand(experts, generator=g)
    for gs in (scales.cuda(), torch.full((experts,), 444.0, device="cuda")):
        out, sf, offsets, position = moe_ffn.dispatch(x, ids, gs)
        want_offsets, row_token, want_position = moe_ffn.plan(ids, experts)
        assert torch.equal(offsets, want_offsets) and torch.equal(position, want_position)
        rows = int(offsets[-1])
        want, want_sf = torch.zeros_like(out), torch.full_like(sf, 0xA5)
        _launcher(quantize, dtype=dtype, in_rows=tokens, rows=tokens * topk, groups=experts, k=hidden)(x, row_token, offsets, want, want_sf, gs)
        assert torch.equal(out[:rows], want[:rows])
        cols = hidden // 16
        group, at = _checks.grouped_sf_rows(offsets, rows)
        assert torch.equal(_checks.logical_scale_bytes(sf, sf.numel() // cols, cols, "128x4")[at],
                           _checks.logical_scale_bytes(want_sf, sf.numel() // cols, cols, "128x4")[at])


@pytest.mark.parametrize("which", [-1, 1, 3, 4])
@pytest.mark.parametrize("sizes", [[0, 0, 5, 0, 130, 1, 0], [257, 0, 31, 33, 128], [1] * 40, [0, 0], [700, 600]], ids=lambda s: "-".join(map(str, s[:8])))
@pytest.mark.parametrize("inner,K,dtype", [(128, 64, "bfloat16"), (384, 704, "float16"), (640, 2048, "bfloat16")])
def test_gated_product_is_product_and_quantizer(which, sizes, inner, K, dtype, variant):
    """The very bytes of the two steps apart: same tiles, same roundings.  (The unfused product runs in the same variant.)"""
    from tirx_kernels import _checks, _native
    from tirx_kernels.basic import moe_ffn, nvfp4_grouped_gemm as product, nvfp4_quantize_grouped as quantize

    rows, groups = max(1, sum(sizes)), len(sizes)
    A, B, SFA, SFB, alpha, offsets, _ = product.prepare_data(rows, groups, 2 * inner, K, bias=False, sizes=sizes)
    gs = 50.0 + 100.0 * torch.rand(groups, device="cuda")
    variant(which)
    out, sf = moe_ffn.gated_product(A, SFA, offsets, B, SFB, alpha, gs, dtype)
    y = torch.zeros(rows, 2 * inner, dtype=getattr(torch, dtype), device="cuda")
    _launcher(product, rows=rows, groups=groups, N=2 * inner, K=K, out_dtype=dtype)(A, B, SFA, SFB, alpha, offsets, None, y)
    want, want_sf = torch.zeros_like(out), torch.zeros_like(sf)
    _launcher(quantize, dtype=dtype, in_rows=rows, rows=rows, groups=groups, k=inner, fuse_silu=True)(y, None, offsets, want, want_sf, gs)
    torch.cuda.synchronize()
    _native.nvfp4_grouped_gemm_status()
    used = sum(sizes)
    assert torch.equal(out[:used], want[:used])
    if used:
        cols = inner // 16
        _, at = _checks.grouped_sf_rows(offsets, used)
        assert torch.equal(_checks.logical_scale_bytes(sf, sf.numel() // cols, cols, "128x4")[at],
                           _checks.logical_scale_bytes(want_sf, sf.numel() // cols, cols, "128x4")[at])


@pytest.mark.parametrize("tokens,topk,n,dtype", [(1, 1, 8, "bfloat16"), (5, 8, 4096, "float16"), (300, 3, 1032, "bfloat16"), (1, 32, 2048, "bfloat16")])
@pytest.mark.parametrize("residual", [False, True])
def test_combine(tokens, topk, n, dtype, residual):
    from tirx_kernels.basic import moe_ffn

    g = torch.Generator().manual_seed(topk)
    rows = max(1, tokens * topk - 2)
    y = torch.randn(rows, n, generator=g).to(getattr(torch, dtype)).cuda()
    position = torch.randint(-2, rows + 2, (tokens, topk), generator=g, dtype=torch.int32).cuda()  # some outside, some twice
    gates = torch.randn(tokens, topk, generator=g).cuda()
    r = torch.randn(tokens, n, generator=g).to(y.dtype).cuda() if residual else None
    live = (position >= 0) & (position < rows)
    terms = y.double()[position.clamp(0, rows - 1).long()] * (gates * live).double()[..., None]
    want = terms.sum(1) + (r.double() if residual else 0)
    size = terms.abs().sum(1) + (r.double().abs() if residual else 0)
    fp32 = (topk + 1) * 2.0**-24 * size  # one rounding per term
    tolerance = torch.finfo(y.dtype).eps / 2 * (want.abs() + fp32) + fp32 + 2.0**-25
    _near(moe_ffn.combine(y, position, gates, r), want, tolerance)
    if residual:
        _near(moe_ffn.combine(y, position, gates, r, out=r), want, tolerance)


# ---- expert feed-forward ----------------------------------------------------------------------------------------------


@pytest.mark.parametrize("tokens,topk,experts,hidden,inner,dtype", [
    (1, 1, 1, 64, 64, "bfloat16"), (1, 8, 8, 256, 128, "float16"), (130, 2, 9, 192, 320, "bfloat16"), (257, 8, 384, 128, 128, "bfloat16"),
    (600, 2, 4, 512, 384, "float16")])
def test_expert_ffn_shapes(tokens, topk, experts, hidden, inner, dtype):
    from tirx_kernels.basic import moe_ffn

    moe_ffn.run_test(tokens, topk, experts, hidden, inner, dtype)


def test_expert_ffn_dropped_repeated_and_residual():
    """An expert named twice counts twice, one that does not exist counts nothing, a token without any keeps its residual."""
    from tirx_kernels.basic import moe_ffn

    x, ids, gates, weights = moe_ffn.prepare_data(6, 4, 8, 256, 128)
    ids = torch.tensor([[1, 1, 2, 3], [-1, -1, -1, -1], [8, 100, 5, 5], [0, 0, 0, 0], [7, 6, 5, 4], [3, -7, 3, 2]], dtype=torch.int32, device="cuda")
    r = torch.randn(6, 256, device="cuda").bfloat16()
    out = moe_ffn.expert_ffn(x, ids, gates, weights, residual=r)
    assert torch.equal(out[1], r[1])
    want = r.double()
    scale = r.double().abs()
    for e in range(8):
        for t, k in torch.nonzero(ids == e).tolist():
            z = moe_ffn._expert(x[t:t + 1], weights, e, "bfloat16")[0] * gates[t, k].double()
            want[t] += z
            scale[t] += z.abs()
    _near(out, want, 2.0**-8 * (want.abs() + scale) + 1e-5)
    assert torch.equal(moe_ffn.expert_ffn(x, ids, gates, weights, residual=r, out=r), out) and torch.equal(r, out)


def test_expert_ffn_zero_tokens():
    from tirx_kernels.basic import moe_ffn

    x, ids, gates, weights = moe_ffn.prepare_data(2, 2, 4, 128, 128)
    assert moe_ffn.expert_ffn(x[:0], ids[:0], gates[:0], weights).shape == (0, 128)


def test_expert_ffn_captured_replayed_and_on_two_streams():
    """Replays follow new inputs and routing; calls on two streams, each with its own workspace, do not meet."""
    from tirx_kernels.basic import moe_ffn

    x, ids, gates, weights = moe_ffn.prepare_data(200, 4, 16, 512, 256)
    want = moe_ffn.expert_ffn(x, ids, gates, weights)
    sx, sids, sg = x.clone(), ids.clone(), gates.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = moe_ffn.expert_ffn(sx, sids, sg, weights)
    order = torch.randperm(200, device="cuda")
    for perm in (torch.arange(200, device="cuda"), order, order.flip(0)):
        sx.copy_(x[perm]), sids.copy_(ids[perm]), sg.copy_(gates[perm])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[perm])
    streams = [torch.cuda.Stream() for _ in range(2)]
    halves = [slice(0, 77), slice(77, 200)]
    expect = [moe_ffn.expert_ffn(x[h].contiguous(), ids[h].contiguous(), gates[h].contiguous(), weights) for h in halves]
    torch.cuda.synchronize()
    got = [[], []]
    inputs = [(x[h].contiguous(), ids[h].contiguous(), gates[h].contiguous()) for h in halves]
    torch.cuda.synchronize()
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(moe_ffn.expert_ffn(*inputs[i], weights))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, expect[i]) for o in got[i])


@pytest.mark.parametrize("tokens,topk,experts,hidden,inner", [(1, 8, 64, 1024, 256), (3, 2, 8, 512, 192), (128, 4, 16, 512, 256), (700, 4, 40, 256, 128)])
def test_expert_ffn_weights_and_routing_written_just_before(tokens, topk, experts, hidden, inner):
    """The products read weights and routing ahead of the launch in front of them, but never ahead of the call."""
    from tirx_kernels.basic import moe_ffn

    x, ids, gates, weights = moe_ffn.prepare_data(tokens, topk, experts, hidden, inner)
    first = [x, ids, gates] + [getattr(weights, f.name) for f in dataclasses.fields(weights)]
    second = [x.flip(1), experts - 1 - ids, gates.flip(1)] + [t.flip(0) for t in first[3:]]  # other rows, experts and weights
    sets = [first, [t.contiguous() for t in second]]
    want = [moe_ffn.expert_ffn(*s[:3], moe_ffn.ExpertWeights(*s[3:])) for s in sets]
    assert not torch.equal(*want)
    live = [t.clone() for t in first]
    live_weights = moe_ffn.ExpertWeights(*live[3:])

    def turn(i):
        for to, new in zip(live, sets[i]):
            to.copy_(new)
        return moe_ffn.expert_ffn(*live[:3], live_weights)

    for _ in range(15):
        for i in range(2):
            assert torch.equal(turn(i), want[i])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = [turn(i % 2) for i in range(6)]
    for _ in range(5):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, want[i % 2]) for i, o in enumerate(outs))


def test_linear_and_norm_captured_and_replayed():
    from tirx_kernels.basic import gated_add_rmsnorm_fp4quant as norm, nvfp4_gemm_epilogue as mod

    data = mod.prepare_data(100, 256, 512)
    ex = _launcher(mod, M=100, N=256, K=512, activation="gelu")
    x, residual, w_post, gate, w_pre, _ = norm.prepare_data("bfloat16", 100, 256, rows_per_gate=30)
    nex = _launcher(norm, input_dtype="bfloat16", M=100, H=256, quantize=False, rows_per_gate=30)
    D, h, y = (torch.empty(100, 256, dtype=torch.bfloat16, device="cuda") for _ in range(3))

    def step():
        ex(*data, D)
        nex(D, residual, w_post, gate, w_pre, h, y, None, None, 0.5, 1e-6)

    step()
    torch.cuda.synchronize()
    first = y.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    y.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, first)
    residual.neg_()
    graph.replay()
    changed = y.clone()
    step()
    torch.cuda.synchronize()
    assert torch.equal(y, changed) and not torch.equal(changed, first)


# ---- gated residual norm ----------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("M,H", [(1, 16), (3, 512), (9, 528), (2, 4096), (5, 4112), (1300, 1040), (2, 16400), (1, 32768), (1200, 8208)])
@pytest.mark.parametrize("post,gate,quantize", [(True, True, True), (False, True, False), (True, False, False), (False, False, True)])
def test_norm_shapes(dtype, M, H, post, gate, quantize):
    from tirx_kernels.basic import gated_add_rmsnorm_fp4quant as mod

    mod.run_test(dtype, M, H, quantize, M % 2 == 1, max(1, M // 3), post, gate, 1.25, 1e-5)


@pytest.mark.parametrize("M,H", [(4, 256), (2500, 256), (2500, 1024), (1300, 16384)])
@pytest.mark.parametrize("quantize", [False, True])
def test_norm_in_place_and_special_rows(M, H, quantize):
    """residual_out may be residual; an all-zero, an infinite and a NaN row leave the others as they are."""
    from tirx_kernels import _checks
    from tirx_kernels.basic import gated_add_rmsnorm_fp4quant as mod

    x, residual, w_post, gate, w_pre, gs = mod.prepare_data("bfloat16", M, H)
    ex = _launcher(mod, input_dtype="bfloat16", M=M, H=H, quantize=quantize, swizzled=False)

    def call(x, residual, out):
        y = torch.empty(M, H // 2, dtype=torch.uint8, device="cuda") if quantize else torch.empty_like(x)
        sf = torch.empty(M * (H // 16), dtype=torch.uint8, device="cuda") if quantize else None
        ex(x, residual, w_post, gate, w_pre, out, y, sf, gs if quantize else None, 0.75, 1e-6)
        return y, sf

    out = torch.empty_like(x)
    clean, clean_sf = call(x, residual, out)
    aliased = residual.clone()
    y, sf = call(x, aliased, aliased)
    assert torch.equal(aliased, out) and torch.equal(y, clean) and (not quantize or torch.equal(sf, clean_sf))
    x2, r2 = x.clone(), residual.clone()
    x2[0], r2[0] = 0, 0
    x2[1, 7] = float("inf")
    if M > 3:
        x2[2, 5] = float("nan")
    y2, sf2 = call(x2, r2, out)
    torch.cuda.synchronize()
    assert torch.equal(y2[3:], clean[3:])
    if quantize:
        assert (y2[0] & 0x77 == 0).all() and (sf2.view(M, -1)[0] == 0).all()
        assert torch.equal(sf2.view(M, -1)[3:], clean_sf.view(M, -1)[3:])
    else:
        assert (y2[0] == 0).all() and y2[1].isnan().any() and (M <= 3 or y2[2].isnan().all())
    assert (out[0] == 0).all()
    assert _checks.E2M1_TABLE[0] == 0.0


def test_norm_zero_rows_and_refusals():
    from tirx_kernels.basic import gated_add_rmsnorm_fp4quant as mod

    e = torch.empty(0, 64, dtype=torch.bfloat16, device="cuda")
    w = torch.ones(64, dtype=torch.bfloat16, device="cuda")
    _launcher(mod, input_dtype="bfloat16", M=0, H=64, quantize=False)(e, e, None, None, w, e, e, None, None, 1.0, 1e-6)
    x = torch.zeros(4, 64, dtype=torch.bfloat16, device="cuda")
    ex = _launcher(mod, input_dtype="bfloat16", M=4, H=64, quantize=False, rows_per_gate=3)
    with pytest.raises(ValueError, match=r"gate must have shape \(2, 64\)"):
        ex(x, x, None, x, w, x, x, None, None, 1.0, 1e-6)
    with pytest.raises(ValueError, match="32-byte"):
        odd = torch.zeros(4 * 64 + 8, dtype=torch.bfloat16, device="cuda")[8:].view(4, 64)
        ex(odd, x, None, None, w, x, x, None, None, 1.0, 1e-6)


# ---- a run of them together ---------------------------------------------------------------------------------------------


@pytest.mark.parametrize("tokens", [1, 37, 300])
def test_a_block_of_them_together(tokens):
    """Residual stream through two half blocks: norm -> product (GELU) -> quantize -> product with the residual -> norm ->
    experts -> norm, each step against its formula on the very operands it got."""
    from tirx_kernels import _checks, _native
    from tirx_kernels.basic import gated_add_rmsnorm_fp4quant as norm, moe_ffn, nvfp4_gemm_epilogue as linear
    from tirx_kernels.basic.nvfp4_gemm import quantize_operand

    H, F = 512, 1024
    g = torch.Generator().manual_seed(tokens)
    draw = lambda *s, std=1.0: (std * torch.randn(*s, generator=g)).to(torch.bfloat16).cuda()
    x, r = draw(tokens, H), draw(tokens, H)
    w_post, w_pre, gate = 1 + draw(H, std=0.1), 1 + draw(H, std=0.1), draw(1, H, std=0.5)
    gs = torch.tensor([400.0], device="cuda")
    nq = _launcher(norm, input_dtype="bfloat16", M=tokens, H=H, quantize=True, swizzled=True, rows_per_gate=tokens)
    h, a, sfa = torch.empty_like(x), torch.empty(tokens, H // 2, dtype=torch.uint8, device="cuda"), \
        torch.empty(_checks.sf_numel(tokens, H // 16, "128x4"), dtype=torch.uint8, device="cuda")
    nq(x, r, w_post, gate, w_pre, h, a, sfa, gs, 1.0, 1e-6)
    rows = torch.arange(tokens, device="cuda")
    _, want_y = norm.expected(x, r, w_post, gate, w_pre, tokens, 1.0, 1e-6, h=h)
    got_y = _checks.dequantize_rows(a, sfa, rows) / 400.0
    assert (got_y - want_y).norm() / want_y.norm() < 0.13  # E2M1 with 16-wide scales: a tenth of the norm

    def product(a, sfa, w, bias, residual, activation):
        N, K = w.shape
        gsw = 2688.0 / w.float().abs().max()
        B, SFB = quantize_operand(w, gsw)
        data = [a, B, sfa, SFB, (1.0 / (gs * gsw)).reshape(1), bias, residual]
        D, want, tolerance = _linear(tokens, N, K, activation, data=data)
        _near(D, want, tolerance)
        return D

    up = product(a, sfa, draw(F, H, std=0.04), draw(F), None, "gelu")
    a2, sfa2 = quantize_operand(up, gs)
    down = product(a2, sfa2, draw(H, F, std=0.04), None, h, "none")
    weights = moe_ffn.prepare_data(1, 2, 4, H, 256)[3]
    ids = torch.randint(0, 4, (tokens, 2), generator=g, dtype=torch.int32).cuda()
    gates = torch.softmax(torch.randn(tokens, 2, generator=g), -1).cuda()
    out = moe_ffn.expert_ffn(down, ids, gates, weights, residual=down)
    want = down.double()
    scale = want.abs()
    for t in range(0, tokens, max(1, tokens // 7)):
        for k in range(2):
            z = moe_ffn._expert(down[t:t + 1], weights, int(ids[t, k]), "bfloat16")[0] * gates[t, k].double()
            want[t] += z
            scale[t] += z.abs()
        _near(out[t], want[t], 2.0**-8 * (want[t].abs() + scale[t]) + 1e-5)
    nb = _launcher(norm, input_dtype="bfloat16", M=tokens, H=H, quantize=False)
    y = torch.empty_like(out)
    nb(out, down, w_post, None, w_pre, h, y, None, None, 0.9, 1e-6)
    want_h, want_y = norm.expected(out, down, w_post, None, w_pre, 1, 0.9, 1e-6, h=h)
    _near(y, want_y, (2.0**-8 + 4e-6) * want_y.abs() + 1e-7)
    _near(h, want_h, 2.0**-8 * want_h.abs() + 2e-6 * (want_h.abs() + 2 * down.double().abs()) + 1e-7)
    torch.cuda.synchronize()
    _native.nvfp4_grouped_gemm_status()


def test_bound_calls_check_every_tensor_and_follow_stream_and_numbers():
    """The compiled check agrees with the spelled-out one; a given number that is none raises; the current stream is used."""
    from tirx_kernels import _checks, _native
    from tirx_kernels.basic import gated_add_rmsnorm_fp4quant as norm

    spec = _checks.tensor_spec
    check = _native.Launch(None, (spec("a", "float32", (2, 3)), spec("b", "uint8", -1, True)))
    a = torch.zeros(2, 3, device="cuda")
    check(a, None), check(a, torch.zeros(0, dtype=torch.uint8, device="cuda")), check(torch.nn.Parameter(a), None)
    for tensors, message in [((a.t().contiguous().t(), None), "contiguous"), ((a.half(), None), "a must be torch.float32"),
                             ((a.view(3, 2), None), "shape"), ((a, a.byte().cpu()), "b: all tensors must be CUDA"), ((None, None), "a must be a tensor")]:
        with pytest.raises(ValueError, match=message):
            check(*tensors)
    x, residual, w_post, gate, w_pre, _ = norm.prepare_data("bfloat16", 6, 256)
    ex = _launcher(norm, input_dtype="bfloat16", M=6, H=256, quantize=False)
    h, y = torch.empty_like(x), torch.empty_like(x)
    with pytest.raises(TypeError):
        ex(x, residual, w_post, gate, w_pre, h, y, None, None, "0.9", 1e-6)
    ex(x, residual, w_post, gate, w_pre, h, y, None, None, 1, 1e-6)  # an integer is a number too
    want = h.clone()
    ex(x, residual, w_post, gate, w_pre, h, y, None, None, 1.0, 1e-6)
    assert torch.equal(h, want)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        late = torch.empty_like(x)
        torch.cuda._sleep(2_000_000)
        late.copy_(x)
        ex(late, residual, w_post, gate, w_pre, h, y, None, None, 1.0, 1e-6)  # behind the copy, on its stream
    stream.synchronize()
    assert torch.equal(h, want)


@pytest.mark.parametrize("M,N,K,which", [(236, 144, 4928, 2), (16, 2048, 4864, 0), (30, 320, 2624, 0), (500, 200, 7104, 2)])
def test_two_issuers_beside_another_stream(M, N, K, which, variant):
    """Tiles with two MMA-issuing warps while another stream's kernels slow some of their warps: the same bits every time."""
    from tirx_kernels import _native
    from tirx_kernels.basic import gated_add_rmsnorm_fp4quant as norm, nvfp4_gemm_epilogue as mod

    variant(which)
    data = mod.prepare_data(M, N, K, residual=False)
    ex = _launcher(mod, M=M, N=N, K=K, activation="gelu_tanh")
    x, residual, w_post, gate, w_pre, _ = norm.prepare_data("bfloat16", 700, 1024)
    nex = _launcher(norm, input_dtype="bfloat16", M=700, H=1024, quantize=False)
    h, y = torch.empty_like(x), torch.empty_like(x)
    want = torch.empty(M, N, dtype=torch.bfloat16, device="cuda")
    ex(*data, want)
    outs = torch.empty(400, M, N, dtype=torch.bfloat16, device="cuda")
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for out in outs:
        with torch.cuda.stream(streams[0]):
            ex(*data, out)
        with torch.cuda.stream(streams[1]):
            nex(x, residual, w_post, gate, w_pre, h, y, None, None, 1.0, 1e-6)
    torch.cuda.synchronize()
    _native.nvfp4_grouped_gemm_status()
    assert (outs == want).all()
