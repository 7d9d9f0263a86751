"""LinearCache on the host: the tensors it refuses."""
import pytest
import torch

from apertura_amd.tree import LinearCache


def test_wrong_tensors_are_refused():
    x, length = torch.zeros(2, 4, 3, 30, 128, dtype=torch.bfloat16), torch.zeros(4, dtype=torch.int32)
    for args in (([], length), ([x] * 9, length), ([x[0]], length), ([x, x[:, :3]], length), ([x, x[:, :, :, :20]], length),
                 ([x.half()], length), ([x[..., ::2]], length), ([x], length[:3]), ([x], length.long()), ([x], torch.zeros(8, dtype=torch.int32)[::2]),
                 ([x], length)):  # not on a GPU
        with pytest.raises(ValueError):
            LinearCache(*args)
