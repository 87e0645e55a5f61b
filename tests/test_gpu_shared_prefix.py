"""pa_decode_shared_prefix against a float64 decode of every sequence.

The bound of an output (derived, nothing fitted).  With u_p the half step of
the probabilities' type (bf16 2^-8; f16 2^-11, where half-precision queries
meet per-tensor scales), u_o that of the output's, a = sum p |v| and dx the
size of a row's largest logit sum:
  * rounding the probabilities moves the output by at most u_p a, and, where the
    sum is that of the rounded ones (per-tensor scales), by u_p |out| more (f16's
    subnormals by a further 2^-25 max|v| a token: the reference exponent keeps
    the largest sum at 1 or more);
  * a logit is a float32 sum of D products and a few float32 factors: it is
    off by at most (D + 8) 2^-24 dx, and exp2 adds 2^-21; a relative error e of
    every probability moves the output by at most 2 e a;
  * sums of n float32 terms: n 2^-24 a for the values and again for the
    denominator, 8 steps per merge level included in the 2 (n + 64);
  * the output's own rounding: u_o |out|.
"""

from __future__ import annotations

import pytest
import torch

from flydsl_amd import _lib, pa_decode_ps_launch, pa_decode_shared_prefix, prepare_pa_decode_shared_prefix
from oracle import shared_prefix as oracle
from tests._prefix_cases import make_prefix_case
from tests.test_gpu_checked import checked  # noqa: F401 (a fixture)
from tests.test_gpu_native import both

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
U = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}


def to_dev(case):
    return {k: (v.to(DEV) if isinstance(v, torch.Tensor) else v) for k, v in case.items()}


def call(d, out, fn=pa_decode_shared_prefix, **kw):
    return fn(out, d["query"], d["key_cache"], d["value_cache"], d["context_lengths"], d["block_tables"],
              d["prefix_indptr"], d["prefix_lengths"], d["softmax_scale"], d["key_scale"], d["value_scale"], **kw)


def reference(d):
    return oracle.decode(d["query"], d["key_cache"], d["value_cache"], d["block_tables"],
                         d["context_lengths"].tolist(), d["prefix_indptr"].tolist(), d["prefix_lengths"].tolist(),
                         d["softmax_scale"], d["key_scale"], d["value_scale"])


def check(d, out, ref=None):
    want, a, dx = ref or reference(d)
    D, n = d["query"].shape[-1], int(d["context_lengths"].max().clamp_min(0))
    f16 = d["query"].dtype == torch.float16 and d["key_scale"].dim() == 1
    u_p = U[torch.float16] if f16 else U[torch.bfloat16]
    e = (D + 8) * 2.0**-24 * dx + 2.0**-21
    tol = (u_p + 2 * e + 2 * (n + 64) * 2.0**-24) * a + (U[out.dtype] + u_p) * want.abs() + 1e-30
    if f16:
        tol = tol + n * 2.0**-25 * 448 * d["value_scale"].double().max()
    err = (out.double() - want).abs()
    assert bool(torch.isfinite(out.float()).all()), "outputs that are not finite"
    worst = (err / tol).max().item()
    assert worst <= 1.0, f"{worst} of the bound, error {err.max().item()}"


def run(case, out_dtype=None, ref=None):
    d = to_dev(case)
    out = torch.full(d["query"].shape, float("nan"), dtype=out_dtype or d["query"].dtype, device=DEV)
    assert call(d, out) == "ps_shared_prefix"
    check(d, out, ref)
    return d, out


def ragged(p, n, step, start=0):
    return (p, [p + start + step * i for i in range(n)])


CASES = {
    "one_token": dict(groups=[(1, [1])]),
    "prefix_is_all": dict(groups=[(40, [40, 40, 40])]),
    "one_suffix_token": dict(groups=[(64, [65, 65])], page=64),
    "small": dict(groups=[ragged(500, 4, 17, 1)]),
    "odd_prefix_inside_a_page": dict(groups=[ragged(77, 5, 9, 1)], page=32),
    "many_rows": dict(groups=[ragged(700, 70, 3, 1)], heads=32, kv_heads=8),
    "groups_and_loose": dict(groups=[ragged(300, 3, 40, 1), (0, [5, 70]), ragged(129, 9, 1, 1)], loose=[0, 1, 333]),
    "mtp": dict(groups=[ragged(200, 6, 31, 4), ragged(1000, 3, 5, 4)], ql=4, heads=64, kv_heads=4, page=64,
                per_token=True),
    "mtp_empty_rows": dict(groups=[(10, [12, 11, 40])], loose=[2, 0, 1, 4], ql=4, heads=8, kv_heads=2),
    "context_inside_the_prefix": dict(groups=[(300, [301, 100, 20, 300, 0])], ql=2),
    "wide_columns": dict(groups=[ragged(130, 2, 20, 5)], ql=5, heads=120, kv_heads=2, page=16),
    "odd_group": dict(groups=[ragged(333, 7, 50, 1)], heads=21, kv_heads=3, ql=3, page=16),
    "page_1024": dict(groups=[ragged(1500, 5, 300, 1)], page=1024, heads=16, kv_heads=2),
    "plain_values": dict(groups=[ragged(250, 5, 33, 1)], trans=False, page=64),
    "plain_values_16": dict(groups=[ragged(250, 5, 33, 1)], trans=False, per_token=True),
    "d64": dict(groups=[ragged(400, 20, 11, 1)], head=64, heads=16, kv_heads=2),
    "d192": dict(groups=[ragged(400, 20, 11, 1)], head=192, heads=16, kv_heads=2),
    "d256": dict(groups=[ragged(400, 20, 11, 1)], head=256, heads=16, kv_heads=2, per_token=True),
    "one_head": dict(groups=[ragged(900, 40, 2, 1)], heads=1, kv_heads=1),
    "long": dict(groups=[ragged(9000, 6, 700, 1)], heads=16, kv_heads=1, page=64),
    "no_groups": dict(groups=[], loose=[1, 64, 65, 900, 0, 17]),
}


@pytest.mark.parametrize("name", CASES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_against_the_definition(name, dtype):
    print(f"[shared-prefix] {name} {dtype}", flush=True)
    run(make_prefix_case(**CASES[name], dtype=dtype, seed=len(name)))


@pytest.mark.parametrize("out_dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("per_token", [False, True])
def test_output_types(out_dtype, per_token):
    run(make_prefix_case(groups=[ragged(200, 9, 13, 1)], per_token=per_token, seed=4), out_dtype)


@pytest.mark.parametrize("scale", [-0.2, 0.0, 3.0])
def test_softmax_scales(scale):
    """Negative, zero (every visible key the same weight) and large ones."""
    case = make_prefix_case(groups=[ragged(150, 4, 30, 1)], seed=6)
    run(dict(case, softmax_scale=scale))


def test_rising_logits_move_the_reference():
    """Keys that grow along the context: the running maximum moves by more
    than the margin many times."""
    case = make_prefix_case(groups=[ragged(900, 4, 90, 1)], per_token=True, seed=7, poison=False)
    ks, bt = case["key_scale"], case["block_tables"]
    for b in range(4):
        for j, p in enumerate(bt[b, : -(-int(case["context_lengths"][b]) // 16)].tolist()):
            ks[p] = ks[p] / ks[p] * 0.002 * (1 + j)
    run(case)


def test_query_and_output_strides():
    case = make_prefix_case(groups=[ragged(100, 3, 30, 1)], seed=8)
    d = to_dev(case)
    r, hq, D = d["query"].shape
    wide_q = torch.full((r, hq + 3, D + 8), float("nan"), dtype=torch.bfloat16, device=DEV)
    wide_q[:, 1 : hq + 1, :D] = d["query"]
    d["query"] = wide_q[:, 1 : hq + 1, :D]
    wide_o = torch.full((r, hq + 1, D + 4), 7.0, dtype=torch.float32, device=DEV)
    out = wide_o[:, :hq, :D]
    call(d, out)
    check(d, out)
    assert (wide_o[:, hq:] == 7).all() and (wide_o[:, :, D:] == 7).all()


def test_cache_views_and_wide_tables():
    """Keys and values interleaved in one allocation; a table with more
    columns and rows than the batch uses, of which the first column is left
    out."""
    case = make_prefix_case(groups=[ragged(100, 3, 30, 1)], seed=9, extra_cols=5)
    d = to_dev(case)
    kc, vc = d["key_cache"], d["value_cache"]
    both = torch.zeros((kc.shape[0], 2, kc[0].numel()), dtype=torch.uint8, device=DEV)
    both[:, 0], both[:, 1] = kc.view(torch.uint8).flatten(1), vc.view(torch.uint8).flatten(1)
    d["key_cache"] = both[:, 0].unflatten(1, kc.shape[1:]).view(torch.float8_e4m3fn)
    d["value_cache"] = both[:, 1].unflatten(1, vc.shape[1:]).view(torch.float8_e4m3fn)
    bt = d["block_tables"]
    wide = torch.full((bt.shape[0] + 4, bt.shape[1] + 1), 2**30, dtype=torch.int32, device=DEV)
    wide[: bt.shape[0], 1:] = bt
    d["block_tables"] = wide[:, 1:]
    out = torch.empty_like(d["query"])
    call(d, out)
    d["block_tables"] = bt
    check(d, out)


def test_agrees_with_the_paged_decode():
    """The same batch through pa_decode_ps_launch, which knows no prefixes:
    each is within 2e-2 of the definition, as that decode's own tests ask."""
    case = make_prefix_case(groups=[ragged(512, 16, 40, 1)], heads=32, kv_heads=8, seed=10)
    d, out = run(case)
    other = torch.empty_like(out)
    pa_decode_ps_launch(other, d["query"], d["key_cache"], d["value_cache"], d["context_lengths"], None, None,
                        d["softmax_scale"], d["key_scale"], d["value_scale"], block_tables=d["block_tables"])
    assert torch.allclose(out.float(), other.float(), atol=2e-2, rtol=2e-2)


def test_same_bits_each_time_and_prepared():
    case = make_prefix_case(groups=[ragged(3000, 40, 20, 1)], heads=32, kv_heads=8, seed=11)
    d, out = run(case)
    again = torch.empty_like(out)
    p = call(d, again, prepare_pa_decode_shared_prefix)
    for _ in range(3):
        again.zero_()
        p.launch()
        assert torch.equal(again, out)


def test_two_streams():
    cases = [make_prefix_case(groups=[ragged(1500, 12, 30, 1)], heads=32, kv_heads=8, seed=s) for s in (12, 13)]
    ds = [to_dev(c) for c in cases]
    outs = [torch.empty_like(d["query"]) for d in ds]
    refs = [reference(d) for d in ds]
    streams = [torch.cuda.Stream() for _ in ds]
    torch.cuda.synchronize()
    for _ in range(4):
        for d, o, s in zip(ds, outs, streams):
            with torch.cuda.stream(s):
                call(d, o)
    torch.cuda.synchronize()
    for d, o, r in zip(ds, outs, refs):
        check(d, o, r)
    outs[0].zero_()
    call(ds[0], outs[0], stream=streams[1])
    torch.cuda.synchronize()
    check(ds[0], outs[0], refs[0])


def test_captured_graphs():
    """Two captured calls, replayed in turn with eager work between them, on
    lengths that change between replays."""
    cases = [make_prefix_case(groups=[ragged(700, 10, 30, 40)], heads=16, kv_heads=2, seed=s, poison=False)
             for s in (14, 15)]
    ds = [to_dev(c) for c in cases]
    outs = [torch.empty_like(d["query"]) for d in ds]
    for d, o in zip(ds, outs):
        call(d, o)
    torch.cuda.synchronize()
    graphs = []
    for d, o in zip(ds, outs):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            call(d, o)
        graphs.append(g)
    eager = torch.empty_like(outs[0])
    for step in range(3):
        for d, o, g in zip(ds, outs, graphs):
            d["context_lengths"] -= 7 * step
            o.fill_(float("nan"))
            g.replay()
            call(d, eager)
            assert torch.equal(o, eager)
            check(d, o)


def test_empty_batch_and_refusals_on_the_device():
    d = to_dev(make_prefix_case(groups=[ragged(30, 3, 5, 1)], seed=16))
    e = dict(d, query=d["query"][:0], context_lengths=d["context_lengths"][:0],
             prefix_indptr=torch.zeros(1, dtype=torch.int32, device=DEV), prefix_lengths=d["prefix_lengths"][:0])
    assert call(e, torch.empty_like(e["query"])) == "ps_shared_prefix"
    with pytest.raises(ValueError, match="must be on"):
        call(dict(d, prefix_lengths=d["prefix_lengths"].cpu()), torch.empty_like(d["query"]))
    q = torch.empty(d["query"].numel() + 4, dtype=torch.bfloat16, device=DEV)[4:].view(d["query"].shape)
    with pytest.raises(RuntimeError, match="PA_ERR_ALIGN"):
        call(dict(d, query=q), torch.empty_like(d["query"]))


@pytest.mark.parametrize("G", [63, 64, 65, 300])
def test_many_groups(G):
    """Groups on both sides of what one wave plans, some of them empty or of no
    shared token, and sequences before and behind them."""
    lens = [(0 if g % 11 == 3 else 5 + 7 * (g % 13), 0 if g % 7 == 5 else 1 + g % 3) for g in range(G)]
    case = make_prefix_case(groups=[(p if k else 0, [p + 1 + 5 * j for j in range(k)]) for p, k in lens],
                            loose=[40, 0, 90], heads=4, kv_heads=1, head=64, seed=G)
    run(case)


@pytest.mark.parametrize("head,B", [(64, 4096), (128, 4096), (192, 2048), (256, 512)])
def test_most_sequences_and_groups(head, B):
    """As many as a call takes: the whole plan beside the tiles."""
    groups = [(3 + g % 29, [3 + g % 29 + (g + j) % 40 for j in range(4)]) for g in range(B // 4)]
    run(make_prefix_case(groups=groups, heads=2, kv_heads=1, head=head, seed=head, spare_pages=1))


def test_bounds_and_lengths_out_of_range():
    """Group bounds that fall or pass the batch, negative lengths and such past
    a table row count as the nearest ones in range."""
    case = make_prefix_case(groups=[ragged(200, 3, 20, 1), ragged(100, 3, 20, 1)], loose=[50, 60], seed=21,
                            poison=False)
    d = to_dev(case)
    cap = d["block_tables"].shape[1] * 16
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)
    for given, meant in (
        (dict(prefix_indptr=i32(-5, 3, 2), prefix_lengths=i32(200, 50)),
         dict(prefix_indptr=i32(0, 3, 3), prefix_lengths=i32(200, 0))),
        (dict(prefix_indptr=i32(3, 2**31 - 1, 3), prefix_lengths=i32(40, 7)),
         dict(prefix_indptr=i32(3, 8, 8), prefix_lengths=i32(40, 0))),
        (dict(prefix_lengths=i32(-3, -2**31)), dict(prefix_lengths=i32(0, 0))),
        (dict(prefix_lengths=i32(2**31 - 1, 100)), dict(prefix_lengths=i32(cap, 100))),
        (dict(context_lengths=i32(-4, -2**31, 2**31 - 1, 100, 50, 40, 30, 20)),
         dict(context_lengths=i32(0, 0, cap, 100, 50, 40, 30, 20))),
    ):
        e, m = dict(d, **given), dict(d, **meant)
        out = torch.full_like(e["query"], float("nan"))
        call(e, out)
        check(m, out)


@pytest.mark.parametrize("kw", [dict(), dict(heads=32, kv_heads=2), dict(per_token=True), dict(head=64, trans=False)])
def test_shared_tokens_that_no_one_sees(kw):
    """A prefix longer than every context of its group, with NaN behind them
    (a page not written yet); a group whose sequences have all ended."""
    case = make_prefix_case(groups=[(300, [301, 100, 20, 130]), (90, [91, 90])], seed=22, **kw)
    ctx = [0, 100, 20, 130, 0, 0]
    bt, v = case["block_tables"], case["value_cache"].view(torch.uint8)
    for t in range(130, 300):
        p, o = int(bt[0, t // 16]), t % 16
        if v.dim() == 5:
            v[p, :, o // 16, :, o % 16] = 0x7F
        else:
            v[p, :, :, o] = 0x7F
        if kw.get("per_token"):
            case["value_scale"][p, :, o] = float("inf")
            case["key_scale"][p, :, o] = float("nan")
    run(dict(case, context_lengths=torch.tensor(ctx, dtype=torch.int32)))


def test_a_sequence_of_nan_leaves_the_others_alone():
    case = make_prefix_case(groups=[ragged(100, 40, 5, 20)], heads=8, kv_heads=2, seed=23)
    d = to_dev(case)
    want = reference(d)
    own = int(case["block_tables"][7, int(case["context_lengths"][7] - 1) // 16])
    d["value_cache"].view(torch.uint8)[own] = 0x7F
    out = torch.empty_like(d["query"])
    call(d, out)
    assert torch.isnan(out[7].float()).all()
    keep = [r for r in range(40) if r != 7]
    sub = dict(d, query=d["query"][keep])
    check(sub, out[keep], tuple(x[keep] for x in want))


@pytest.mark.parametrize("per_token", [False, True])
def test_offsets_past_32_bits(per_token):
    """Pages more than 4 GiB apart."""
    case = make_prefix_case(groups=[ragged(700, 4, 60, 1)], heads=8, kv_heads=2, per_token=per_token, page=64, seed=24)
    d = to_dev(case)
    nb = d["key_cache"].shape[0]
    step = -(-(5 << 30) // nb) // 1024 * 1024
    big = torch.empty(nb * step, dtype=torch.uint8, device=DEV)
    at = 0
    for name in ("key_cache", "value_cache", "key_scale", "value_scale"):
        t = d[name]
        if t.dim() < 4:
            continue
        raw = t.view(torch.uint8).flatten(1)
        view = big.view(nb, step)[:, at: at + raw.shape[1]]
        view.copy_(raw)
        at += raw.shape[1]
        d[name] = view.view(t.dtype).unflatten(1, t.shape[1:])
    assert d["key_cache"].stride(0) == step and (nb - 1) * step > 1 << 32
    out = torch.empty_like(d["query"])
    call(d, out)
    check({**to_dev(case)}, out)


@pytest.mark.parametrize("kw", [
    dict(groups=[ragged(300, 5, 30, 1)], loose=[70]),
    dict(groups=[ragged(300, 5, 30, 4)], ql=4, heads=16, kv_heads=2, per_token=True, dtype=torch.float16, page=64),
    dict(groups=[ragged(200, 3, 30, 1)], trans=False, head=64),
    dict(groups=[], loose=[5, 6]),
])
def test_native_path_gives_the_same_bits(monkeypatch, kw):
    d = to_dev(make_prefix_case(**kw, seed=25))

    def both_ways():
        out = torch.full_like(d["query"], 3.0)
        return call(d, out), out

    both(monkeypatch, both_ways)


@pytest.mark.parametrize("kw", [dict(heads=8, kv_heads=2), dict(heads=32, kv_heads=2),
                                dict(heads=8, kv_heads=2, per_token=True)])
def test_checked_build(checked, kw):
    """Clean calls note nothing; table entries outside the cache are read as the
    nearest page and noted."""
    case = make_prefix_case(groups=[ragged(200, 6, 40, 1)], loose=[90], seed=26, poison=False, **kw)
    run(case)
    assert _lib.debug_violations(checked) == 0
    bt, nb = case["block_tables"].clone(), case["key_cache"].shape[0]
    bt[0, 3], bt[4, 14], bt[6, 2] = -9, nb + 5, 2**31 - 1
    d = to_dev(dict(case, block_tables=bt))
    out = torch.empty_like(d["query"])
    call(d, out)
    check(dict(d, block_tables=d["block_tables"].clamp(0, nb - 1)), out)
    assert _lib.debug_violations(checked) == _lib.VIOLATION_PAGE


def test_scales_and_caches_in_other_forms():
    """Scales left out or given as numbers, caches as bytes: the same bits as
    tensors of one value and fp8 caches."""
    d = to_dev(make_prefix_case(groups=[ragged(100, 3, 30, 1)], seed=27))
    one = torch.ones(1, device=DEV)
    want, got = (torch.empty_like(d["query"]) for _ in range(2))
    call(dict(d, key_scale=one, value_scale=one), want)
    call(dict(d, key_scale=None, value_scale=None), got)
    assert torch.equal(got, want)
    call(dict(d, key_scale=1.0, value_scale=one, key_cache=d["key_cache"].view(torch.uint8),
              value_cache=d["value_cache"].view(torch.uint8), softmax_scale=d["softmax_scale"]), got)
    assert torch.equal(got, want)
    call(dict(d, key_scale=one, value_scale=one, softmax_scale=0), got)  # a whole number
    call(dict(d, key_scale=one, value_scale=one, softmax_scale=0.0), want)
    assert torch.equal(got, want)
