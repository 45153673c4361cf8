"""GPU parity of the feed-forward operators: every module's own configurations against its 64-bit formula."""

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
