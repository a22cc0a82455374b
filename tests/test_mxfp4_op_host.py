"""What xv::mxfp4_linear, the op that a compiler's trace of mxfp4_linear holds,
refuses, without a GPU: the launch is replaced, so that a call that gets as far
fails its test instead of running."""
import pytest
import torch

from xvllm.layers.linear import mxfp4_linear


@pytest.fixture(autouse=True)
def no_launch(monkeypatch):
    import xvllm._torch_glue as glue

    def launched(name, device, *args):
        raise AssertionError(f"{name} launched for device {device}")

    monkeypatch.setattr(glue, "call", launched)


def _operands(m=3, n=8, k=64):
    return (torch.zeros(m, k, dtype=torch.bfloat16), torch.zeros(n, k // 2, dtype=torch.uint8),
            torch.zeros(n, k // 32, dtype=torch.uint8))


@pytest.mark.parametrize("silu", [False, True])
def test_compiled_function_refuses_cpu_tensors(silu):
    x, w, s = _operands()
    w, s = w.view(torch.float4_e2m1fn_x2), s.view(torch.float8_e8m0fnu)
    with pytest.raises(RuntimeError, match="GPU"):
        mxfp4_linear(x, w, s, silu_mul=silu)
    f = torch.compile(lambda t: mxfp4_linear(t, w, s, silu_mul=silu), backend="eager", fullgraph=True)
    with torch.no_grad(), pytest.raises(RuntimeError, match="GPU"):
        f(x)


def test_raw_op_refuses_what_the_function_refuses():
    op = torch.ops.xv.mxfp4_linear
    x, w, s = _operands()
    with pytest.raises(RuntimeError, match="GPU"):
        op(x, w, s, False)
    for bad in ((x[:, :32], w, s), (x, w[:, :16], s), (x, w, s[:, :1]), (x, w[:4], s), (x, w, s[:4]), (x[:, :48], w[:, :24], s[:, :1]),
                (x[None], w, s), (x[0], w, s), (x, w[0], s), (x[:, :0], w[:, :0], s[:, :0])):
        with pytest.raises(ValueError):
            op(*bad, False)
    with pytest.raises(ValueError, match="even"):
        op(x, w[:7], s[:7], True)
    for bad in ((x.float(), w, s), (x, w.float(), s), (x, w, s.to(torch.int32))):
        with pytest.raises(TypeError):
            op(*bad, False)
    wide = torch.zeros(8, 40, dtype=torch.uint8)
    for bad in ((x, wide[:, :32], s), (x, w[:1].expand(8, 32), s), (x, torch.zeros(32, 8, dtype=torch.uint8).t(), s),
                (x, w, s[:1].expand(8, 2)), (x, w, torch.zeros(2, 8, dtype=torch.uint8).t())):
        with pytest.raises(ValueError, match="in place"):
            op(*bad, False)


class _On(torch.Tensor):
    """A CPU tensor that says it is on a GPU."""

    device_index = 0

    def get_device(self):
        return self.device_index


def _on(t, index):
    t = t.as_subclass(_On)
    t.device_index = index
    return t


def test_product_refuses_operands_of_several_devices():
    from xvllm.layers.linear import _mxfp4_product

    for at in ((0, 1, 0), (0, 0, 1), (1, 0, 0), (0, -1, 0), (0, 0, -1), (-1, 0, 0)):
        with pytest.raises(RuntimeError, match="one device"):
            _mxfp4_product(*(_on(t, i) for t, i in zip(_operands(), at)), False)
    x, w, s = _operands()
    w = torch.zeros(8 * 32 + 8, dtype=torch.uint8)[8:].view(8, 32)
    with pytest.raises(ValueError, match="aligned"):
        _mxfp4_product(_on(x, 0), _on(w, 0), _on(s, 0), False)
