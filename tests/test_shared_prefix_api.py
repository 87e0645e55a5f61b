"""The float64 oracle of the shared-prefix decode against the brute force,
and the launcher's checks, on the CPU."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import flydsl_amd.shared_prefix as sp
from flydsl_amd import _lib, prepare_pa_decode_shared_prefix
from oracle import np_ref, shared_prefix
from tests._prefix_cases import make_prefix_case


class StubStream:
    cuda_stream = 0


@pytest.fixture(autouse=True)
def no_device(monkeypatch):
    monkeypatch.setattr(sp, "_cu_count", lambda device=None: 256)


def prep(case, **kw):
    d = dict(case, **kw)
    out = d.pop("output", None)
    if out is None:
        out = torch.empty_like(d["query"])
    return prepare_pa_decode_shared_prefix(
        out, d["query"], d["key_cache"], d["value_cache"], d["context_lengths"], d["block_tables"],
        d["prefix_indptr"], d["prefix_lengths"], d["softmax_scale"], d["key_scale"], d["value_scale"],
        stream=StubStream())


@pytest.mark.parametrize("kw", [
    dict(groups=[(20, [21, 30]), (5, [6])], loose=[0, 9], page=16, heads=4, kv_heads=2, head=64),
    dict(groups=[(33, [35, 40, 34])], page=32, ql=2, heads=4, kv_heads=1, head=64, per_token=True, trans=False),
])
def test_oracle_against_brute_force(kw):
    c = make_prefix_case(**kw, dtype=torch.float16, seed=1)
    out, a, dx = shared_prefix.decode(
        c["query"], c["key_cache"], c["value_cache"], c["block_tables"], c["context_lengths"].tolist(),
        c["prefix_indptr"].tolist(), c["prefix_lengths"].tolist(), c["softmax_scale"], c["key_scale"],
        c["value_scale"])
    pt = c["key_scale"].dim() > 1
    want = np_ref.paged_decode_f64(
        c["query"].float().numpy(), c["key_cache"].view(torch.uint8).numpy(), c["value_cache"].view(torch.uint8).numpy(),
        c["block_tables"].numpy(), c["context_lengths"].numpy(), kw.get("ql", 1), c["softmax_scale"],
        c["key_scale"].numpy() if pt else float(c["key_scale"]),
        c["value_scale"].numpy() if pt else float(c["value_scale"]))
    assert np.abs(out.numpy() - want).max() < 1e-12
    assert (a >= out.abs() - 1e-12).all() and (dx >= 0).all()


def test_marshalling():
    c = make_prefix_case(groups=[(100, [120, 130, 101])], loose=[7], ql=1, heads=8, kv_heads=2, page=32,
                         per_token=True, extra_cols=2)
    a = prep(c).args
    assert (a.num_seqs, a.num_groups, a.num_kv_heads, a.query_length, a.query_group_size) == (4, 1, 2, 1, 4)
    assert (a.head_size, a.block_size, a.per_token_kv, a.trans_v, a.num_workers) == (128, 32, 1, 1, 512)
    assert a.num_blocks == c["key_cache"].shape[0] and a.max_blocks_per_seq == c["block_tables"].shape[1]
    assert a.stride_bt_seq == c["block_tables"].stride(0) and a.stride_ks_block == 64 and a.stride_ks_head == 32
    assert a.prefix_indptr == c["prefix_indptr"].data_ptr() and a.prefix_lengths == c["prefix_lengths"].data_ptr()
    assert prep(c).route == "ps_shared_prefix"


def test_refusals():
    c = make_prefix_case(groups=[(100, [120, 130, 101])], page=32)

    def bad(match, err=ValueError, **kw):
        with pytest.raises(err, match=match):
            prep(c, **kw)

    i32 = lambda *x: torch.tensor(x, dtype=torch.int32)
    bad("must have 3 dimensions", query=c["query"][0])
    bad("output shape", output=torch.empty(3, 8, 64))
    bad("Unsupported output dtype", output=torch.empty(3, 8, 128, dtype=torch.float64))
    bad("Unsupported query dtype", query=c["query"].float())
    bad("only supports bf16/f16", query=c["query"].to(torch.float8_e4m3fn))
    bad("multiple of the batch", context_lengths=i32(5, 6))
    bad("divisible by KV heads", query=c["query"][:, :7], output=c["query"][:, :7].clone())
    bad("head_dim=96", NotImplementedError, query=torch.empty(3, 8, 96, dtype=torch.bfloat16))
    bad("page size", key_cache=c["key_cache"][..., :24, :])
    bad("key_cache must be", key_cache=c["key_cache"][:, :, :4])
    bad("value_cache must be", value_cache=c["value_cache"][:, :1])
    bad("fp8 e4m3fn", key_cache=c["key_cache"].view(torch.int8))
    bad("contiguous within", key_cache=c["key_cache"].view(torch.uint8).transpose(2, 3).contiguous().transpose(2, 3))
    bad("last dimension", block_tables=c["block_tables"].t().contiguous().t())
    bad("must be int32", prefix_lengths=c["prefix_lengths"].long())
    bad("must be contiguous", context_lengths=i32(1, 2, 3, 4, 5, 6)[::2])
    bad("prefix_indptr must have 2", prefix_indptr=i32(0, 1, 2))
    bad("rows for 3 sequences", block_tables=c["block_tables"][:2])
    bad("at least one page", block_tables=c["block_tables"][:, :0])
    bad("both hold one value", key_scale=torch.ones(2))
    bad("per-token scales", key_scale=torch.ones(c["key_cache"].shape[0], 2, 32, 1))
    many = torch.zeros(5000, dtype=torch.int32)
    bad("at most 4096", NotImplementedError, query=torch.empty(5000, 8, 128, dtype=torch.bfloat16),
        context_lengths=many, block_tables=many[:, None])
    wide = make_prefix_case(groups=[(10, [12])], head=256, page=32)
    with pytest.raises(NotImplementedError, match="at most 512"):
        prep(wide, query=torch.empty(513, 8, 256, dtype=torch.bfloat16), context_lengths=many[:513],
             block_tables=many[:513, None])
    with pytest.raises(RuntimeError, match="must be on a GPU"):
        prepare_pa_decode_shared_prefix(torch.empty_like(c["query"]), *[c[k] for k in (
            "query", "key_cache", "value_cache", "context_lengths", "block_tables", "prefix_indptr", "prefix_lengths",
            "softmax_scale", "key_scale", "value_scale")])


def test_c_entry_refuses_before_any_launch():
    lib = _lib.load()
    assert lib.pa_fp8_decode_shared_prefix(None, None, 0, None) == -1
    a = _lib.SharedPrefixArgs()
    rc = lambda n=1 << 40: lib.pa_fp8_decode_shared_prefix(a, 4096, n, None)
    a.abi_version = 99
    assert rc() == -8
    a.abi_version = _lib.ABI_VERSION
    for f in ("output", "query", "key_cache", "value_cache", "block_tables", "context_lengths", "prefix_indptr",
              "prefix_lengths", "key_scale", "value_scale"):
        setattr(a, f, 4096)  # aligned stand-ins that nothing here reads
    a.num_seqs, a.num_groups, a.num_kv_heads, a.query_length, a.query_group_size = 4, 1, 2, 1, 4
    a.head_size, a.block_size, a.num_blocks, a.max_blocks_per_seq, a.num_workers = 128, 16, 8, 4, 256
    need = _lib.shared_prefix_workspace_bytes(4, 1, 2, 1, 4, 128, 256)
    assert rc(need - 1) == -9
    for field, value, code in (("head_size", 96, -2), ("block_size", 24, -3), ("block_size", 2048, -3),
                               ("block_size", 8, -3), ("num_seqs", 4097, -6), ("num_groups", 1025, -6),
                               ("num_blocks", 0, -6), ("max_blocks_per_seq", 0, -6), ("query_dtype", 2, -5),
                               ("output_dtype", 3, -5), ("query", None, -1), ("prefix_lengths", None, -1),
                               ("query", 4104, -7), ("stride_q_tok", 4, -7), ("stride_k_block", 8, -7),
                               ("stride_out_head", 2, -7), ("num_workers", 0, -6)):
        old = getattr(a, field)
        setattr(a, field, value)
        assert rc(need - 1) == code, (field, value)
        setattr(a, field, old)
    a.num_seqs = 0
    assert rc(0) == 0  # nothing to do
