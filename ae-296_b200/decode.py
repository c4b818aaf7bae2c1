"""The operators around the delta in a decode step.

* :func:`int4_linear`       the base projection with 4-bit weights that the delta is added to;
* :func:`append_kv`         what the layer does with q, k, v and their deltas next: add, rotate by position, write k and v
                            to a paged cache;
* :func:`prefix_attention`  attention of one query token per request over that cache, in which groups of neighbouring
                            requests share a prefix.  In a multi-LoRA server k and v depend on the adapter, so those
                            that can share one are the requests of an adapter
                            (:func:`ae296_b200.batching.prefix_groups`).

Like the other ops these are one C-ABI call each (``include/b200_decode.h``) through the native host path; the checks
here name what is wrong with a call that it does not take.  All tensors of a call are on one device, and the work is
enqueued on that device's current stream.  Nothing is kept between calls.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _lib
from ._lib import check
from .ops import _require_cuda

# bits of a `status` word; the last: a wait inside a kernel ran out, and the outputs concerned are NaN
BAD_SLOT, BAD_POSITION, BAD_PAGE, BAD_LENGTH, BAD_GROUPS, TIMEOUT = 1, 2, 4, 8, 16, 32


def _refuse(what: str, tests) -> None:
    """Raises for the first of ``(condition, reason)`` that does not hold; a condition may rely on those before it."""
    for ok, why in tests:
        if not ok():
            raise ValueError(f"{what}: {why}")
    raise ValueError(f"{what}: unsupported arguments")


def _same_device(what: str, required, optional) -> None:
    present = [*required, *(t for t in optional if t is not None)]
    if not all(isinstance(t, torch.Tensor) for t in present):
        raise ValueError(f"{what}: tensors expected")
    _require_cuda(*present)
    if len({t.device for t in present}) != 1:
        raise ValueError(f"{what}: all tensors must be on one device")


def _cache_tests(k_cache, v_cache, q):
    return [
        (lambda: q.dim() == 3, "q must be [tokens, heads, head_dim]"),
        (lambda: q.dtype in (torch.float16, torch.bfloat16), "fp16 or bf16 tensors expected"),
        (lambda: k_cache.dim() == 4 and k_cache.shape == v_cache.shape, "the caches must be [pages, page_size, kv_heads, head_dim]"),
        (lambda: k_cache.numel() > 0, "the cache is empty"),
        (lambda: k_cache.stride() == v_cache.stride() and k_cache.stride(3) == 1,
         "the two caches must have the same strides, and contiguous heads"),
        (lambda: k_cache.dtype == q.dtype and v_cache.dtype == q.dtype, "q and the caches must have one type"),
        (lambda: q.shape[-1] == k_cache.shape[-1], "q and the cache differ in head_dim"),
    ]


def _status_test(status):
    return (lambda: status is None or (status.dtype == torch.int32 and status.numel() == 1), "status must be one int32")


def append_kv(q_out: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor,
              v_cache: torch.Tensor, positions: torch.Tensor, slots: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
              dq: Optional[torch.Tensor] = None, dk: Optional[torch.Tensor] = None, dv: Optional[torch.Tensor] = None,
              interleaved: bool = False, status: Optional[torch.Tensor] = None) -> None:
    """``q_out = rot(q + dq)``, ``k_cache[slot] = rot(k + dk)``, ``v_cache[slot] = v + dv`` for every token, in one launch.

    ``q``, ``q_out`` and ``dq`` are ``[T, heads, D]``, ``k``, ``v``, ``dk`` and ``dv`` ``[T, kv_heads, D]``, with any strides over tokens
    and heads (parts of one fused product, for instance); ``dq``, ``dk``, ``dv`` are the LoRA deltas that the layer code
    otherwise adds first (lightllm/models/llama/layer_infer/transformer_layer_infer.py:160-170).  The caches are one
    layer's ``[pages, page_size, kv_heads, D]``, both with the same strides (the reference's table of token slots,
    lightllm/common/mem_manager.py:28-38, is one of pages of 1).  ``slots [T]`` says where a token goes (``page * page_size +
    place``), ``positions [T]`` which row of ``cos`` and ``sin`` ``[positions, R/2]`` (fp32, or the type of q) it is turned by; both int32 or int64.
    The first ``R`` elements of a head turn, in pairs ``(i, i + R/2)``, or ``(2i, 2i + 1)`` when ``interleaved``.  Sums and products are fp32,
    rounded once.  ``q_out`` may be ``q``.

    A token with a negative slot is padding: nothing of it is written, neither to the cache nor to ``q_out``.  One whose
    slot lies behind the cache, or whose position lies outside the tables, is left out too and sets ``BAD_SLOT`` or
    ``BAD_POSITION`` in ``status`` (one int32 on the device, for the caller to clear and to read).  The slots of a call differ."""
    rc = _lib.host().append_kv(q_out, q, k, v, k_cache, v_cache, positions, slots, cos, sin, dq, dk, dv, interleaved, status)
    if rc > 0:
        _same_device("append_kv", (q_out, q, k, v, k_cache, v_cache, positions, slots, cos, sin), (dq, dk, dv, status))
        deltas = [("dq", dq, q), ("dk", dk, k), ("dv", dv, v)]
        _refuse("append_kv", _cache_tests(k_cache, v_cache, q) + [
            (lambda: q_out.shape == q.shape, "q_out must have q's shape"),
            (lambda: k.dim() == 3 and v.dim() == 3 and k.shape == v.shape, "k and v must be [tokens, kv_heads, head_dim]"),
            (lambda: k.shape[0] == q.shape[0] and tuple(k.shape[1:]) == tuple(k_cache.shape[2:]), "q, k, v and the cache disagree in shape"),
            (lambda: all(t.dtype == q.dtype for t in (q_out, k, v)), "q_out, q, k and v must have one type"),
        ] + [(lambda d=d, x=x: d is None or (d.shape == x.shape and d.dtype == x.dtype), f"{name} must have the shape and type of what it is added to")
             for name, d, x in deltas] + [
            (lambda: all(t is None or t.stride(2) == 1 for t in (q_out, q, k, v, dq, dk, dv)), "heads must be contiguous"),
            (lambda: positions.dim() == 1 and slots.dim() == 1 and positions.shape[0] == slots.shape[0] == q.shape[0] and
             positions.is_contiguous() and slots.is_contiguous(), "positions and slots must be contiguous [tokens]"),
            (lambda: positions.dtype in (torch.int32, torch.int64) and slots.dtype in (torch.int32, torch.int64), "positions and slots must be int32 or int64"),
            (lambda: cos.dim() == 2 and cos.shape == sin.shape and cos.stride() == sin.stride() and cos.stride(1) == 1 and cos.shape[0] > 0,
             "cos and sin must be [positions, R/2] with the same strides"),
            (lambda: 0 < 2 * cos.shape[1] <= q.shape[2], "the tables turn more elements than a head has, or none"),
            (lambda: cos.dtype == sin.dtype and cos.dtype in (torch.float32, q.dtype), "cos and sin must be fp32 or of q's type"),
            _status_test(status)])
    check(rc, "append_kv")


def prefix_attention(out: torch.Tensor, q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
                     lens: torch.Tensor, prefix_table: Optional[torch.Tensor] = None, prefix_lens: Optional[torch.Tensor] = None,
                     group_starts: Optional[torch.Tensor] = None, scale: Optional[float] = None, lse: Optional[torch.Tensor] = None,
                     status: Optional[torch.Tensor] = None) -> None:
    """``out[b] = softmax(scale * q[b] K^T) V`` over the keys of ``b``'s group's prefix followed by its own; one query token per request.

    ``q`` and ``out`` are ``[B, heads, D]``, the caches one layer's ``[pages, page_size, kv_heads, D]`` (``D`` 64 or 128, ``page_size`` a power of
    two up to 256, both caches with the same strides, 16-byte aligned); query head ``h`` reads cache head ``h // (heads // kv_heads)``.  Request ``b``'s own
    keys are the first ``lens[b]`` of the pages ``block_table[b]`` (int32 ``[B, M]``).  Group ``g`` holds the requests ``group_starts[g]`` to
    ``group_starts[g + 1] - 1`` and its prefix is the first ``prefix_lens[g]`` keys of the pages ``prefix_table[g]`` (int32 ``[G, M']``): they are read
    once for all the group's requests.  Requests in no group, and all of them without the three arguments, have no prefix.
    ``scale`` defaults to ``D ** -0.5``.  ``lse`` (fp32 ``[B, heads]``) receives the natural logarithm of the sum of exponentials, with which
    results over further keys can be joined.

    A request without any key gets zeros and ``lse`` -inf.  Whatever the cache holds behind the lengths, NaN included, has no
    influence.  Lengths and tables stay on the device; a page outside the cache is left out, a length outside its table is cut,
    group starts that do not ascend inside the batch leave all prefixes out; each sets its bit (``BAD_PAGE``, ``BAD_LENGTH``,
    ``BAD_GROUPS``; ``TIMEOUT`` if a wait inside the kernel ran out) in ``status`` (one int32 on the device, for the caller to clear and to read).  At most 4096 requests and 2048 groups."""
    rc = _lib.host().prefix_attention(out, q, k_cache, v_cache, block_table, lens, prefix_table, prefix_lens, group_starts, scale, lse, status)
    if rc > 0:
        _same_device("prefix_attention", (out, q, k_cache, v_cache, block_table, lens), (prefix_table, prefix_lens, group_starts, lse, status))
        given = [x is not None for x in (prefix_table, prefix_lens, group_starts)]
        i32 = [t for t in (block_table, lens, prefix_table, prefix_lens, group_starts) if t is not None]
        tests = _cache_tests(k_cache, v_cache, q) + [
            (lambda: out.shape == q.shape and out.dtype == q.dtype, "out must have q's shape and type"),
            (lambda: q.stride(2) == 1 and out.stride(2) == 1, "heads must be contiguous"),
            (lambda: q.shape[2] in (64, 128), "head_dim must be 64 or 128"),
            (lambda: q.shape[1] % k_cache.shape[2] == 0 and q.shape[1] <= 1024, "heads must be a multiple of kv_heads, at most 1024"),
            (lambda: q.shape[0] <= 4096, "at most 4096 requests"),
            (lambda: all(t.dtype == torch.int32 for t in i32), "tables, lengths and group starts must be int32"),
            (lambda: block_table.dim() == 2 and block_table.shape[0] == q.shape[0] and (block_table.stride(1) == 1 or block_table.shape[1] <= 1),
             "block_table must be [requests, pages] with contiguous rows"),
            (lambda: lens.dim() == 1 and lens.shape[0] == q.shape[0] and lens.is_contiguous(), "lens must be contiguous [requests]"),
            (lambda: all(given) or not any(given), "prefix_table, prefix_lens and group_starts go together"),
            (lambda: scale is None or hasattr(scale, "__float__"), "scale must be a number")]
        if all(given):
            tests += [
                (lambda: prefix_table.dim() == 2 and prefix_table.shape[0] <= 2048, "at most 2048 groups"),
                (lambda: (prefix_table.stride(1) == 1 or prefix_table.shape[1] <= 1), "prefix_table must be [groups, pages] with contiguous rows"),
                (lambda: prefix_lens.dim() == 1 and prefix_lens.shape[0] == prefix_table.shape[0] and prefix_lens.is_contiguous(), "prefix_lens must be contiguous [groups]"),
                (lambda: group_starts.dim() == 1 and group_starts.shape[0] == prefix_table.shape[0] + 1 and group_starts.is_contiguous(), "group_starts must be contiguous [groups + 1]")]
        _refuse("prefix_attention", tests + [
            (lambda: lse is None or (lse.dtype == torch.float32 and tuple(lse.shape) == tuple(q.shape[:2]) and lse.is_contiguous()),
             "lse must be contiguous fp32 [requests, heads]"),
            _status_test(status)])
    check(rc, "prefix_attention")


def int4_linear(y: torch.Tensor, x: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor, zeros: Optional[torch.Tensor] = None,
                add: Optional[torch.Tensor] = None, status: Optional[torch.Tensor] = None) -> None:
    """``y = x W^T (+ add)`` with ``W[n, k] = scales[n, k // group] * (code[n, k] - zero[n, k // group])``, for the few tokens of a decode step.

    ``x [T, K]``, ``y [T, N]`` (x's type, or fp32), ``codes`` uint8 ``[N, K/2]`` (column ``2i`` in the low four bits of byte ``i``, ``2i + 1`` in the high ones),
    ``scales [N, K/group]`` of x's type, ``zeros`` uint8 of the same shape (0..15; without them 8 everywhere), ``add [T, N]`` of y's type, which may be
    ``y``.  ``group`` (32, 64 or 128) follows from the shapes.  Rows of x, y and add may be strided; x and the codes start at 16-byte
    boundaries, x's rows too.  The sums are fp32 and rounded once.  Should a wait inside the kernel run out, the outputs concerned are NaN and
    ``TIMEOUT`` is set in ``status`` (one int32 on the device, for the caller to clear and to read)."""
    rc = _lib.host().int4_linear(y, x, codes, scales, zeros, add, status)
    if rc > 0:
        _same_device("int4_linear", (y, x, codes, scales), (zeros, add, status))
        _refuse("int4_linear", [
            (lambda: x.dim() == 2 and y.dim() == 2 and codes.dim() == 2 and scales.dim() == 2, "x, y, codes and scales must be matrices"),
            (lambda: x.dtype in (torch.float16, torch.bfloat16), "x must be fp16 or bf16"),
            (lambda: y.dtype in (x.dtype, torch.float32), "y must be of x's type or fp32"),
            (lambda: codes.dtype == torch.uint8 and 2 * codes.shape[1] == x.shape[1], "codes must be uint8 [outputs, inputs / 2]"),
            (lambda: scales.shape[1] > 0 and x.shape[1] / scales.shape[1] in (32, 64, 128), "the group must be 32, 64 or 128 columns"),
            (lambda: scales.dtype == x.dtype and scales.shape[0] == codes.shape[0], "scales must be [outputs, groups] of x's type"),
            (lambda: tuple(y.shape) == (x.shape[0], codes.shape[0]), "y must be [tokens, outputs]"),
            (lambda: x.stride(1) == 1 and y.stride(1) == 1, "rows of x and y must be contiguous"),
            (lambda: codes.is_contiguous() and scales.is_contiguous(), "codes and scales must be contiguous"),
            (lambda: zeros is None or (zeros.dtype == torch.uint8 and zeros.shape == scales.shape and zeros.is_contiguous()),
             "zeros must be contiguous uint8 of the scales' shape"),
            (lambda: add is None or (add.dtype == y.dtype and add.shape == y.shape and add.stride(1) == 1), "add must have y's shape and type"),
            _status_test(status)])
    check(rc, "int4_linear")
