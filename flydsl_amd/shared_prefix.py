"""Decode attention of a batch whose sequences share prefixes.

:func:`pa_decode_shared_prefix` gives what
:func:`flydsl_amd.pa_decode_ps_launch` gives on the same query, caches, block
tables and context lengths, and reads the tokens that a group of sequences
shares once for the whole group (flydsl_amd/csrc/shared_prefix.hip).  It has
no counterpart in the reference; layouts, scales, dtypes and errors follow
pa_decode_ps_launch (kernels/pa_decode_fp8.py:2812-3202).

Groups: sequences ``prefix_indptr[g] .. prefix_indptr[g + 1] - 1`` have the same
first ``prefix_lengths[g]`` tokens, as sequences forked off one prompt have
(:func:`flydsl_amd.fork_cache_pages`).  They are read through the block-table
row of the group's first sequence, which has to hold their pages whatever its
own context length; the tokens behind them through each sequence's own row.
The shared length need not end with a page.  Sequences before, between (groups
of length 0) and behind the groups are decoded by themselves.
"""

from __future__ import annotations

import ctypes

import torch

from . import _lib
from ._lib import DTYPE_BF16, DTYPE_F16
from .pa_decode import (
    _check_int32,
    _cu_count,
    _get_output_dtype_code,
    _get_query_input_dtype,
    _is_current_stream_capturing,
    _prepare_scale_tensor,
)

ROUTE = "ps_shared_prefix"
HEAD_SIZES = (64, 128, 192, 256)
MAX_SEQS = {64: 4096, 128: 4096, 192: 2048, 256: 512}  # by head size; a quarter as many groups


def _workers(device) -> int:
    """Persistent workgroups of a launch: two fit a compute unit."""
    return 2 * _cu_count(device)


class PreparedSharedPrefix:
    """A validated call with its C-ABI arguments marshalled; ``launch()``
    issues it.  The tensors must stay alive and unchanged in shape; launches
    of one prepared call share its workspace, so they must not overlap."""

    def __init__(self, args, stream, device, keepalive):
        self.route = ROUTE
        self.args = args
        self._keep = keepalive
        self._lib = None
        if stream is None:  # an empty batch: nothing to launch
            return
        self._lib = _lib.load()
        self._device = device
        self._stream = ctypes.c_void_p(stream.cuda_stream)
        n = _lib.shared_prefix_workspace_bytes(args.num_seqs, args.num_groups, args.num_kv_heads, args.query_length,
                                               args.query_group_size, args.head_size, args.num_workers)
        # allocated on the call's stream, so that its memory's next use comes
        # after the launches
        s = stream
        if not isinstance(stream, torch.cuda.Stream):
            s = torch.cuda.ExternalStream(stream.cuda_stream, device) if device.type == "cuda" else None
        with torch.cuda.stream(s):
            self._workspace = torch.empty(n, dtype=torch.uint8, device=device)

    def launch(self) -> str:
        if self._lib is not None:
            with torch.cuda.device(self._device):
                rc = self._lib.pa_fp8_decode_shared_prefix(ctypes.byref(self.args), self._workspace.data_ptr(),
                                                           self._workspace.numel(), self._stream)
            _lib.check(rc, "pa_fp8_decode_shared_prefix")
        return self.route


def pa_decode_shared_prefix(
    output: torch.Tensor,
    query: torch.Tensor,
    key_cache: torch.Tensor,
    value_cache: torch.Tensor,
    context_lengths: torch.Tensor,
    block_tables: torch.Tensor,
    prefix_indptr: torch.Tensor,
    prefix_lengths: torch.Tensor,
    softmax_scale: float,
    key_scale: torch.Tensor = None,
    value_scale: torch.Tensor = None,
    *,
    stream=None,
) -> str:
    """FP8 paged decode that reads shared prefixes once.

    output, query [B*ql, Hq, D] (output bf16/f16/f32, query bf16/f16);
    key_cache [NB, Hkv, D/16, bs, 16] and value_cache [NB, Hkv, bs/16, D, 16]
    (or [NB, Hkv, D, bs]) fp8 e4m3fn; context_lengths [B] (all tokens of a
    sequence, the prefix among them); block_tables [B, max_blocks]; prefix_indptr
    [G+1] and prefix_lengths [G] int32 on the device.  key/value_scale: float,
    [1] tensor or [NB, Hkv, bs, 1].  Query token i of a sequence of n tokens
    sees keys 0 .. n - ql + i; a row that sees none is zero.  head_dim 64,
    128, 192 or 256, page size 16 to 1024 (a power of two), any query_length x
    group size, up to 4096 sequences and 1024 groups (head_dim 192: 2048 and 512;
    256: 512 and 128).  Returns the route name.
    Under graph capture the scales must be float32 device tensors.
    """
    native = _lib.native()
    if native is not None and stream is None and native.shared_prefix(
            output, query, key_cache, value_cache, context_lengths, block_tables, prefix_indptr, prefix_lengths,
            softmax_scale, key_scale, value_scale, _workers):
        return ROUTE
    return prepare_pa_decode_shared_prefix(
        output, query, key_cache, value_cache, context_lengths, block_tables, prefix_indptr, prefix_lengths,
        softmax_scale, key_scale, value_scale, stream=stream).launch()


def prepare_pa_decode_shared_prefix(
    output: torch.Tensor,
    query: torch.Tensor,
    key_cache: torch.Tensor,
    value_cache: torch.Tensor,
    context_lengths: torch.Tensor,
    block_tables: torch.Tensor,
    prefix_indptr: torch.Tensor,
    prefix_lengths: torch.Tensor,
    softmax_scale: float,
    key_scale: torch.Tensor = None,
    value_scale: torch.Tensor = None,
    *,
    stream=None,
) -> PreparedSharedPrefix:
    """Validate and marshal one call (arguments and errors of
    :func:`pa_decode_shared_prefix`)."""
    dev = query.device
    capturing = _is_current_stream_capturing()
    for name, t, dims in (("query", query, (3,)), ("output", output, (3,)), ("key_cache", key_cache, (5,)),
                          ("value_cache", value_cache, (4, 5)), ("context_lengths", context_lengths, (1,)),
                          ("block_tables", block_tables, (2,)), ("prefix_indptr", prefix_indptr, (1,)),
                          ("prefix_lengths", prefix_lengths, (1,))):
        if t.dim() not in dims:
            raise ValueError(f"`{name}` must have {' or '.join(map(str, dims))} dimensions, got {tuple(t.shape)}")
        if t.device != dev:
            raise ValueError(f"`{name}` must be on {dev}, got {t.device}")
    key_scale = _prepare_scale_tensor("key_scale", key_scale, device=dev, is_graph_capturing=capturing)
    value_scale = _prepare_scale_tensor("value_scale", value_scale, device=dev, is_graph_capturing=capturing)
    dtype = _get_query_input_dtype(query)
    if dtype == "packed_fp8":
        raise ValueError("`pa_decode_shared_prefix` only supports bf16/f16 query inputs")
    out_dtype = _get_output_dtype_code(output)
    rows, hq, d = query.shape
    nb, hkv, bs = int(key_cache.shape[0]), int(key_cache.shape[1]), int(key_cache.shape[3])
    b, g = int(context_lengths.shape[0]), int(prefix_lengths.shape[0])
    ql = rows // b if b else 0
    if ql * b != rows or (b and not ql):
        raise ValueError(f"query rows ({rows}) must be a positive multiple of the batch size ({b})")
    if hkv == 0 or hq == 0 or hq % hkv:
        raise ValueError("Query heads must be divisible by KV heads")
    if d not in HEAD_SIZES:
        raise NotImplementedError(f"head_dim={d} is not built; pa_decode_shared_prefix supports {HEAD_SIZES}")
    if bs not in (16, 32, 64, 128, 256, 512, 1024):
        raise ValueError(f"page size must be a power of two in [16, 1024], got {bs}")
    if tuple(key_cache.shape[2:]) != (d // 16, bs, 16):
        raise ValueError(f"key_cache must be [NB, Hkv, {d // 16}, bs, 16], got {tuple(key_cache.shape)}")
    trans_v = value_cache.dim() == 5
    want = (nb, hkv, bs // 16, d, 16) if trans_v else (nb, hkv, d, bs)
    if tuple(value_cache.shape) != want:
        raise ValueError(f"value_cache must be {list(want)}, got {list(value_cache.shape)}")
    for name, t in (("key_cache", key_cache), ("value_cache", value_cache)):
        if t.dtype not in (torch.float8_e4m3fn, torch.uint8):
            raise ValueError(f"`{name}` must be fp8 e4m3fn (or its bytes as uint8), got {t.dtype}")
        if nb and not t[0, 0].is_contiguous():
            raise ValueError(f"`{name}` must be contiguous within a page's head")
    for name, t in (("query", query), ("output", output), ("block_tables", block_tables)):
        if t.stride(-1) != 1:
            raise ValueError(f"`{name}` must be contiguous in its last dimension")
    if tuple(output.shape) != tuple(query.shape):
        raise ValueError(f"output shape {tuple(output.shape)} must match query shape {tuple(query.shape)}")
    per_token = key_scale.dim() > 1
    if per_token:
        if tuple(key_scale.shape) != (nb, hkv, bs, 1) or tuple(value_scale.shape) != (nb, hkv, bs, 1):
            raise ValueError(f"per-token scales must be [NB, Hkv, bs, 1], got {tuple(key_scale.shape)} and "
                             f"{tuple(value_scale.shape)}")
        if key_scale.stride() != value_scale.stride() or key_scale.stride(2) != 1:
            raise ValueError("key_scale and value_scale must share strides with a contiguous token dimension")
    elif value_scale.dim() > 1 or key_scale.numel() != 1 or value_scale.numel() != 1:
        raise ValueError("key_scale and value_scale must both hold one value, or both be [NB, Hkv, bs, 1]")
    for name, t in (("context_lengths", context_lengths), ("block_tables", block_tables),
                    ("prefix_indptr", prefix_indptr), ("prefix_lengths", prefix_lengths)):
        _check_int32(name, t, dev)
    for name, t in (("context_lengths", context_lengths), ("prefix_indptr", prefix_indptr),
                    ("prefix_lengths", prefix_lengths)):
        if not t.is_contiguous():
            raise ValueError(f"`{name}` must be contiguous")
    if block_tables.shape[0] < b:
        raise ValueError(f"block_tables has {block_tables.shape[0]} rows for {b} sequences")
    if prefix_indptr.shape[0] != g + 1:
        raise ValueError(f"prefix_indptr must have {g + 1} entries for {g} groups, got {prefix_indptr.shape[0]}")
    if b > MAX_SEQS[d] or g > MAX_SEQS[d] // 4:
        raise NotImplementedError(f"at most {MAX_SEQS[d]} sequences and {MAX_SEQS[d] // 4} groups with head_dim={d}, got "
                                  f"{b} and {g}")

    a = _lib.SharedPrefixArgs()
    if b == 0:
        return PreparedSharedPrefix(a, None, dev, ())
    if nb == 0 or block_tables.shape[1] == 0:
        raise ValueError("the cache and the block tables must hold at least one page")
    if dev.type != "cuda" and stream is None:
        raise RuntimeError("pa_decode_shared_prefix: tensors must be on a GPU (the decode runs only in libpa_fp8.so)")
    a.abi_version = _lib.ABI_VERSION
    a.output, a.query = output.data_ptr(), query.data_ptr()
    a.key_cache, a.value_cache = key_cache.data_ptr(), value_cache.data_ptr()
    a.block_tables, a.context_lengths = block_tables.data_ptr(), context_lengths.data_ptr()
    a.prefix_indptr = prefix_indptr.data_ptr()
    a.prefix_lengths = prefix_lengths.data_ptr() if g else None
    a.key_scale, a.value_scale = key_scale.data_ptr(), value_scale.data_ptr()
    a.stride_q_tok, a.stride_q_head = query.stride(0), query.stride(1)
    a.stride_k_block, a.stride_k_head = key_cache.stride(0), key_cache.stride(1)
    a.stride_v_block, a.stride_v_head = value_cache.stride(0), value_cache.stride(1)
    a.stride_bt_seq = block_tables.stride(0)
    if per_token:
        a.stride_ks_block, a.stride_ks_head = key_scale.stride(0), key_scale.stride(1)
    a.stride_out_tok, a.stride_out_head = output.stride(0), output.stride(1)
    a.num_seqs, a.num_groups, a.num_kv_heads = b, g, hkv
    a.query_length, a.query_group_size, a.head_size = ql, hq // hkv, d
    a.block_size, a.num_blocks, a.max_blocks_per_seq = bs, nb, int(block_tables.shape[1])
    a.per_token_kv, a.trans_v = int(per_token), int(trans_v)
    a.query_dtype = DTYPE_BF16 if dtype == "bf16" else DTYPE_F16
    a.output_dtype = out_dtype
    a.num_workers = _workers(dev)
    a.softmax_scale = float(softmax_scale)
    keep = (output, query, key_cache, value_cache, context_lengths, block_tables, prefix_indptr, prefix_lengths,
            key_scale, value_scale)
    return PreparedSharedPrefix(a, stream if stream is not None else torch.cuda.current_stream(dev), dev, keep)
