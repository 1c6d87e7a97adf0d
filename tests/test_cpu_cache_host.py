"""A paged cache in host memory is refused by the launchers that take its device from it (no GPU)."""
import pytest
import torch

import redline_amd as ra
from redline_amd import kernels as K


def test_a_cache_on_the_cpu_is_refused():
    kv = K.KVCache(1, 4, 2, 64, device="cpu").layer(0)
    f16, i32, f32 = (lambda *s, d=d: torch.zeros(*s, dtype=d) for d in (torch.float16, torch.int32, torch.float32))
    for n in (0, 4):
        with pytest.raises(ra.Error, match="GPU tensors"):
            K.rope_and_write_kv_norm(f16(4, 512), i32(4), i32(4), n, 4, f32(8, 32), f32(8, 32), kv)
        with pytest.raises(ra.Error, match="GPU tensors"):
            K.read_kv(kv, i32(4), n, f16(4, 128), f16(4, 128))
