"""The qwen3 recipe's 8-bit precision against its mesh: refused when the configuration is validated."""

import pytest

from recipes.qwen3.configs.schema import Qwen3Config


def config(precision, **mesh):
    return {"model": {"linear_precision": precision}, "parallel": {"mesh": mesh}}


@pytest.mark.parametrize("mesh", [{"tensor": 2}, {"context": 4}, {"shard": 1, "tensor": 2, "context": 2}])
def test_refused_with_tensor_or_context_parallelism(mesh):
    with pytest.raises(ValueError, match="linear_precision"):
        Qwen3Config.model_validate(config("fp8", **mesh))
    Qwen3Config.model_validate(config("bf16", **mesh))


@pytest.mark.parametrize("mesh", [{}, {"shard": 1}, {"replicate": 2, "shard": 4}, {"tensor": 1, "context": 1}])
def test_accepted_on_data_parallel_meshes(mesh):
    assert Qwen3Config.model_validate(config("fp8", **mesh)).model.linear_precision == "fp8"


def test_unknown_precision_is_refused():
    with pytest.raises(ValueError):
        Qwen3Config.model_validate(config("int8"))
