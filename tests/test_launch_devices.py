"""Which operands the binding's launch context takes: tensors of one GPU, and nothing else, in whatever order they come.
Stand-ins for the tensors, so that no GPU is needed; nothing is launched."""

import itertools

import pytest
import torch


class _Operand:
    """What the context looks at of a tensor."""

    def __init__(self, device):
        self.device = torch.device(device)
        self.is_cuda = self.device.type == "cuda"

    def get_device(self):
        return self.device.index if self.is_cuda else -1


KINDS = [None, "cpu", "meta", "cuda:0", "cuda:1"]


@pytest.mark.parametrize("count", [0, 1, 2, 3, 4])
def test_operands_are_on_one_gpu_in_every_order(count):
    from cute_kernels import _C

    for kinds in itertools.product(KINDS, repeat=count):
        operands = [None if kind is None else _Operand(kind) for kind in kinds]
        devices = {kind for kind in kinds if kind is not None}
        if len(devices) == 1 and devices <= {"cuda:0", "cuda:1"}:
            assert _C._Launch(*operands).index == int(devices.pop()[-1]), kinds
            assert _C._require_gpu(*operands).type == "cuda"
            continue
        with pytest.raises(RuntimeError, match="need GPU tensors|on different devices|no tensor"):
            _C._Launch(*operands)
            pytest.fail(f"taken: {kinds}")
        with pytest.raises(RuntimeError):
            _C._require_gpu(*operands)


def test_real_host_tensors_are_refused_in_front_of_a_gpu_tensor():
    from cute_kernels import _C

    host = torch.zeros(4)
    for operands in [(host,), (host, _Operand("cuda:0")), (None, host, host, _Operand("cuda:0")),
                     (_Operand("cuda:0"), host), (host.to("meta"), _Operand("cuda:0"))]:
        with pytest.raises(RuntimeError, match="need GPU tensors"):
            _C._Launch(*operands)
