"""The overlap of two tensors' rows that the norm and the fp8 quantisers go by, against sets of their bytes."""
import random

import torch

from gsp._native import rows_meet


def _view(rng, buffer):
    while True:
        flat = buffer.view(rng.choice([torch.uint8, torch.int16]))
        rows, width, pitch = rng.randint(0, 6), rng.randint(1, 20), rng.choice([0, 5, 10, 16, 16, 24, 24, 32, 40])
        first = rng.randint(0, 100)
        if first + max(0, rows - 1) * pitch + width <= flat.numel():
            return torch.as_strided(flat, (rows, width), (pitch, 1), first)


def _bytes(t):
    size = t.element_size()
    return {(t.storage_offset() + i * t.stride(0)) * size + k for i in range(t.shape[0]) for k in range(t.shape[1] * size)}


def test_rows_meet():
    rng, buffer = random.Random(1), torch.zeros(400, dtype=torch.uint8)
    found = [0, 0]
    for _ in range(20000):
        a, b = _view(rng, buffer), _view(rng, buffer)
        want = bool(_bytes(a) & _bytes(b))
        assert rows_meet(a, b) == rows_meet(b, a) == want, (a.shape, a.stride(), a.storage_offset(), a.dtype, b.shape,
                                                            b.stride(), b.storage_offset(), b.dtype)
        found[want] += 1
    assert min(found) > 1000
