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
