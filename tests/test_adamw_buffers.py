"""What AdamW and AdamW8bit allocate does not follow torch's default dtype:
device buffers that the kernels read and write as fp32 are fp32."""

import pytest
import torch
from torch.overrides import TorchFunctionMode

from smo_optimizer_b200 import AdamW, AdamW8bit, _lib, grad_norm

HYPER_BYTES = _lib.ADAMW_HYPER_DTYPE.itemsize


class _CudaAsMeta(TorchFunctionMode):
    """Tensors made on a CUDA device are made without memory instead."""

    def __torch_function__(self, func, types, args=(), kwargs=None):
        kwargs = dict(kwargs or {})
        if kwargs.get("device") is not None and torch.device(kwargs["device"]).type == "cuda":
            kwargs["device"] = "meta"
        return func(*args, **kwargs)


@pytest.fixture(params=[torch.bfloat16, torch.float16, torch.float32, torch.float64], ids=str)
def default_dtype(request):
    kept = torch.get_default_dtype()
    torch.set_default_dtype(request.param)
    yield request.param
    torch.set_default_dtype(kept)


@pytest.mark.parametrize("cls", [AdamW, AdamW8bit])
def test_scalar_and_norm_buffers_are_fp32(cls, default_dtype):
    opt = cls([torch.nn.Parameter(torch.zeros(10))], capturable=True, max_grad_norm=1.0)
    with _CudaAsMeta():
        opt._scalar_address(0, 40)
        max_norm, _, _, nbytes = opt._norm_buffers(0, 40)
    scalars, (workspace, norm) = opt._scalars[0], opt._workspace[0]
    assert scalars.dtype == torch.float32 and scalars.numel() * scalars.element_size() == 40 * HYPER_BYTES
    assert norm.dtype == torch.float32 and norm is opt.last_grad_norm
    assert workspace.dtype == torch.uint8 and workspace.numel() == nbytes and max_norm == 1.0


@pytest.mark.parametrize("cls", [AdamW, AdamW8bit])
def test_states_and_step_counts_are_fp32(cls, default_dtype):
    p = torch.nn.Parameter(torch.zeros(5000, dtype=torch.bfloat16))
    opt = cls([p], capturable=True)
    opt._init_state(p, opt.param_groups[0])
    st = opt.state[p]
    assert st["step"].dtype == torch.float32
    floats = {k: t.dtype for k, t in st.items() if k in ("exp_avg", "exp_avg_sq", "m_s", "v_s")}
    assert len(floats) == 2 and set(floats.values()) == {torch.float32}
    for step in (1001, 1001.0, torch.tensor(1001.0, dtype=torch.float64), torch.tensor([1001])):
        got = opt._step_value(p, step)
        assert got.dtype == torch.float32 and got.shape == () and float(got) == 1001.0


def test_norm_without_gradients_is_an_fp32_zero_on_the_cpu(default_dtype):
    got = grad_norm([torch.nn.Parameter(torch.zeros(3))])
    assert got.dtype == torch.float32 and got.device.type == "cpu" and float(got) == 0.0
