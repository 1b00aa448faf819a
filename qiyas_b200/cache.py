"""A cache of keys and values in 8 bits: int8 codes with one f32 scale for each block, a block being a page of consecutive
tokens of one sequence in one head.  ``GpuOps.CacheWrite``, ``CacheRead`` and ``CacheAttention`` work on it; the reference
has no counterpart (it keeps keys and values in its plain types).

``BlockCache`` holds the four device arrays:

========  ======================================  ============================================================
k_codes   int8 [pages, heads, page, dim]          page: 16, 32, 64 or 128 tokens; dim: a multiple of 16 up to 256
v_codes   int8 [pages, heads, page, dim]
k_scales  float32 [pages, heads]                  a stored value is code * scale, any finite number
v_scales  float32 [pages, heads]
========  ======================================  ============================================================

Which pages belong to which sequence is the caller's: an int32 table [sequences, width] on the device, entry [b, i] naming
the page that holds tokens i * page .. i * page + page - 1 of sequence b.
"""
import torch

from . import _lib

PAGES = (16, 32, 64, 128)
_INT8, _F32 = torch.int8, torch.float32


class BlockCache:
    """The arrays of a cache, checked once; nothing is copied."""

    def __init__(self, k_codes, v_codes, k_scales, v_scales):
        shape, pairs = k_codes.shape, k_scales.shape
        if len(shape) != 4 or v_codes.shape != shape:
            raise ValueError(f"codes are [pages, heads, page, dim] twice: got {tuple(shape)}, {tuple(v_codes.shape)}")
        self.pages, self.heads, self.page, self.dim = pages, heads, page, dim = shape
        if pairs != (pages, heads) or v_scales.shape != pairs:
            raise ValueError(f"scales are [pages, heads] = {(pages, heads)}: got {tuple(pairs)}, {tuple(v_scales.shape)}")
        if page not in PAGES or dim % 16 or not 0 < dim <= 256:
            raise NotImplementedError(f"blocks of {page} tokens x {dim}: 16, 32, 64 or 128 tokens, and dim a multiple of 16 up to 256")
        self.index = index = k_codes.get_device()               # -1: not on a GPU
        if not (k_codes.dtype is v_codes.dtype is _INT8 and k_scales.dtype is v_scales.dtype is _F32 and k_codes.is_contiguous()
                and v_codes.is_contiguous() and k_scales.is_contiguous() and v_scales.is_contiguous()
                and v_codes.get_device() == k_scales.get_device() == v_scales.get_device() == index):
            raise ValueError("contiguous int8 codes and float32 scales on one device are needed, got " +
                             ", ".join(f"{t.dtype} {t.stride()} on {t.device}" for t in (k_codes, v_codes, k_scales, v_scales)))
        self.k_codes, self.v_codes, self.k_scales, self.v_scales = k_codes, v_codes, k_scales, v_scales
        self.parts = _lib.CACHE(k_codes.data_ptr(), v_codes.data_ptr(), k_scales.data_ptr(), v_scales.data_ptr(), pages, heads, page, dim)

    @classmethod
    def empty(cls, pages, heads, page, dim, device="cuda:0"):
        """A cache of `pages` pages; nothing in it needs initialising."""
        codes = [torch.empty(pages, heads, page, dim, dtype=torch.int8, device=device) for _ in range(2)]
        scales = [torch.empty(pages, heads, dtype=torch.float32, device=device) for _ in range(2)]
        return cls(*codes, *scales)

    @property
    def nbytes(self):
        return 2 * self.pages * self.heads * (self.page * self.dim + 4)


__all__ = ["BlockCache", "PAGES"]
