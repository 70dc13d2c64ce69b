"""What the fine-tuning operators refuse at the ends of their ranges, found on the host."""
import importlib

import pytest

torch = pytest.importorskip("torch")


class OnDevice:
    """A tensor's outside: `n` elements at an address of device `dev`."""

    def __init__(self, n, dtype=torch.float32, dev=0):
        self.n, self.dtype, self.dev, self.device, self.is_cuda = n, dtype, dev, f"cuda:{dev}", True

    def numel(self):
        return self.n

    def is_contiguous(self):
        return True

    def get_device(self):
        return self.dev

    def data_ptr(self):
        return 0x7f0000000000


@pytest.mark.parametrize("other", ["param", "grad", "copy", "exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale"])
def test_adamw_refuses_tensors_of_another_device(jc, monkeypatch, other):
    training = importlib.import_module("julia-cuda_b200.training")
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    state = torch.float8_e4m3fn
    t = {"param": OnDevice(300), "grad": OnDevice(300, torch.bfloat16), "copy": OnDevice(300, torch.float16),
         "exp_avg": OnDevice(300, state), "exp_avg_sq": OnDevice(300, state), "exp_avg_scale": OnDevice(2),
         "exp_avg_sq_scale": OnDevice(2)}
    t[other].dev = 1
    states = {k: [v] for k, v in t.items() if k.startswith("exp")}
    with pytest.raises(jc.JuliaCudaError, match="on the current device"):
        training.AdamW([t["param"]], [t["grad"]], bits=8, copies=[t["copy"]], **states)


@pytest.mark.parametrize("rows", [2 ** 31, 2 ** 32 - 1])
def test_more_rows_than_the_kernels_count(jc, rows):
    """Rows are walked with 32-bit counters that pass the last row by up to a grid's step."""
    L, p = jc.lib(), 4096
    assert L.jc_layer_norm(0, p, 1, p, p, 1e-5, rows, 1, p, 1, None, None) == -1 and "2^31 - 1" in jc.last_error()
    assert L.jc_layer_norm_backward(0, p, 1, p, 1, p, p, None, 0, rows, 1, p, 1, p, p, p, None) == -1
    assert "2^31 - 1" in jc.last_error()
    assert L.jc_layer_norm_ws_floats(rows, 1) >= 148 * 2

    def linear(m, n, k):
        return L.jc_linear(0, 0, p, k, p, k, None, None, n, p, n, None, n, m, n, k, p, None)

    def backward(m, n, k):
        return L.jc_linear_backward(0, 0, p, n, p, k, p, k, None, n, m, n, k, p, k, p, k, p, p, None)
    for call in (linear, backward):
        for size in ((rows, 16, 16), (16, rows, 16), (16, 16, rows)):
            assert call(*size) == -1 and "2^31 - 1" in jc.last_error(), (size, jc.last_error())


def test_tensors_with_more_rows_than_the_kernels_count(jc):
    x, v = torch.empty(2 ** 31, 1, dtype=torch.float16, device="meta"), torch.empty(1, device="meta")
    for call in (lambda: jc.layer_norm(x, v, None, x), lambda: jc.layer_norm_backward(x, x, v, v, x),
                 lambda: jc.linear(x, x, x), lambda: jc.linear_backward(x, x, x, dx=x)):
        with pytest.raises(jc.JuliaCudaError, match="2\\^31 - 1"):
            call()
