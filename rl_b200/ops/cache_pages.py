"""Copies of KV-cache pages.

Counterpart: the block copies of the paged caches that the reference's rollout engines keep
(vLLM / MCore dynamic inference, ``block_size_tokens: 256``,
``examples/configs/grpo_math_1B.yaml:345``).  Here one kernel (``csrc/cache_pages.cu``) copies any
list of pages in every layer, K and V, at once: whole pages when a prompt is given to the other
rows of its group, the filled part of the last page when a row is forked.
"""

from __future__ import annotations

from typing import Optional, Sequence, Union

import torch

from rl_b200.ops._ext import add_launches, ext, use_native

__all__ = ["copy_cache_pages"]

_Ints = Union[Sequence[int], torch.Tensor]


def _host_ints(name: str, x: _Ints) -> list[int]:
    if isinstance(x, torch.Tensor):
        if x.is_cuda:
            raise ValueError(f"copy_cache_pages: {name} must be host data (a list or a CPU tensor)")
        if x.is_floating_point() or x.dtype == torch.bool or x.dim() != 1:
            raise ValueError(f"copy_cache_pages: {name} must be a vector of integers, got {tuple(x.shape)} {x.dtype}")
        return x.tolist()
    return list(x)


def _check_pages(src, dst, tokens, pages, block) -> tuple[int, int]:
    """The checks of the native call (which makes its own): (kind, position) of the first fault."""
    written: set = set()
    for i, (a, b, t) in enumerate(zip(src, dst, tokens)):
        if not (0 <= a < pages and 0 <= b < pages):
            return 1, i
        if not 0 <= t <= block:
            return 2, i
        if b in written:
            return 3, i
        written.add(b)
    return next(((4, i) for i, a in enumerate(src) if a in written), (0, 0))


def copy_cache_pages(cache: torch.Tensor, src: _Ints, dst: _Ints, tokens: Optional[_Ints] = None) -> None:
    """Copy the first ``tokens[i]`` tokens (default: all) of page ``src[i]`` to page ``dst[i]``,
    in place, in every layer of ``cache [..., pages, block, kv heads, head dim]`` (contiguous, any type).

    ``src``, ``dst`` and ``tokens`` are host data.  A page may be copied to many, but a page that is
    written may neither be written twice nor be a source (``ValueError``); page numbers outside the
    cache raise ``IndexError``.  Tokens behind ``tokens[i]`` of a destination keep their values.
    """
    if cache.dim() < 4 or not cache.is_contiguous():
        raise ValueError("copy_cache_pages: a contiguous cache [..., pages, block, kv heads, head dim] expected, got "
                         f"{tuple(cache.shape)}")
    pages, block = cache.shape[-4], cache.shape[-3]
    s, d = _host_ints("src", src), _host_ints("dst", dst)
    n = [block] * len(s) if tokens is None else _host_ints("tokens", tokens)
    if not len(s) == len(d) == len(n):
        raise ValueError(f"copy_cache_pages: {len(s)} sources, {len(d)} destinations, {len(n)} token counts")
    planes = cache.view(-1, pages, block, cache.shape[-2] * cache.shape[-1]) if cache.numel() else None
    if use_native(cache) and planes is not None:
        bad, i = ext().copy_cache_pages(planes, s, d, n)
        if not bad:
            add_launches(i)
    else:
        bad, i = _check_pages(s, d, n, pages, block)
    if bad == 1:
        raise IndexError(f"copy_cache_pages: page {s[i]} -> {d[i]} of a cache of {pages} pages")
    if bad:
        raise ValueError("copy_cache_pages: " + {2: f"{n[i]} tokens of a page of {block}",
                                                 3: f"page {d[i]} is written twice",
                                                 4: f"page {s[i]} is both read and written"}[bad])
    if cache.is_cuda:
        return
    if planes is None:
        return
    raw = planes.view(torch.uint8) if planes.element_size() == 1 else planes  # fp8 caches: the bytes
    for a, b, t in zip(s, d, n):
        raw[:, b, :t] = raw[:, a, :t]
