"""The `torch.webgpu` device module.

`is_initialized` and `current_device` are what the reference provides
(python/torch_webgpu/webgpu/__init__.py:1-9); the rest is what torch's generic
device plumbing (seeding, `torch.get_device_module`) and users of a real GPU
backend look for.
"""
import struct

import torch

from .. import _C

__all__ = [
    "is_initialized", "current_device", "device_count", "is_available", "init", "synchronize",
    "empty_cache", "memory_stats", "get_device_name", "get_device_properties", "manual_seed_all",
    "manual_seed", "initial_seed", "get_rng_state", "set_rng_state", "device", "get_amp_supported_dtype",
]


# torch.utils.checkpoint saves and restores the generator's state on devices that say this, so that a
# recomputed dropout drops what the forward pass dropped.
_initialized = True


class device:
    """`with torch.webgpu.device(0):` there is one device, which is always the current one."""

    def __init__(self, device=None):
        index = device if isinstance(device, int) or device is None else torch.device(device).index
        if index not in (None, -1, 0):
            raise ValueError(f"webgpu has a single device, got index {index}")

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        return False


def get_amp_supported_dtype():
    """No op of this backend is autocast; torch asks before it enters a (disabled) autocast region."""
    return []


def init():
    """Bind the GPU and create the stream now instead of at first use."""
    _C._init()


def is_initialized():
    return bool(_C._is_initialized())


def is_available():
    try:
        _C._init()
        return True
    except RuntimeError:
        return False


def current_device():
    return 0


def device_count():
    return 1


def synchronize(device=None):
    """Wait until every queued kernel and copy has finished."""
    _C._synchronize()


def empty_cache():
    """Return cached, unused device blocks to the driver."""
    _C._empty_cache()


def memory_stats(device=None):
    return _C._memory_stats()


def get_device_properties(device=None):
    return _C._device_info()


def get_device_name(device=None):
    return _C._device_info()["name"]


# What draws random numbers on the device is dropout.  Its generator is counter-based: a seed, and
# an offset that every call takes one of; torch.manual_seed() sets it through these hooks.
def _is_in_bad_fork():
    return False


def manual_seed_all(seed):
    """Seed dropout's generator and start its offsets at 0 (torch.manual_seed() does this)."""
    _C._set_rng_state(int(seed) & (2 ** 64 - 1), 0)


def manual_seed(seed):
    manual_seed_all(seed)


def initial_seed():
    return _C._get_rng_state()[0]


def get_rng_state(device=None):
    """The generator's seed and next offset as 16 bytes."""
    return torch.tensor(list(struct.pack("<QQ", *_C._get_rng_state())), dtype=torch.uint8)


def set_rng_state(new_state, device=None):
    """Put the generator back to what get_rng_state returned."""
    if new_state.dtype != torch.uint8 or new_state.numel() != 16:
        raise ValueError("expected the 16 bytes that get_rng_state returns")
    _C._set_rng_state(*struct.unpack("<QQ", bytes(new_state.tolist())))
