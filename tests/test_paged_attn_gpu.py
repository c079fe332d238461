"""The paged full-attention calls on the GPU against their 64-bit statement (operators_ref):
append, decode step, prompt attention. Tolerances, derived:
  append   the value rounded to bf16: half a step, 2^-8 of it, and fp32 arithmetic before it (the
           norm's sum of 256, the rotation): 2e-6 of the head's largest value
  step     fp32 output: fp32 sums of head_dim products (2^-24 sqrt(256) of sum |q k|), exp2 at 2^-22,
           sums over the positions: 2e-5 of the largest sum of p |v|; bf16 output: 2^-8 of the value
           and the two-part products' residue, 2^-16 of the scores (up to 2 reach) and of p |v|
  prefill  bf16 output: 2^-8 of the value; p rounded to bf16: 2^-8 of the sum of p |v|; q rounded to
           bf16: a score off by 2^-8 sum |q k| scale (reach), so a normalised weight by twice that;
           and, over all outputs, three roundings of 2^-8 / sqrt(3) at most in the 2-norm"""
import numpy as np
import pytest
import torch

import nmoe_b200 as N
from operators_ref import Packed

pytestmark = pytest.mark.gpu
H = 2.0 ** -8

# (q heads, KV heads, head dim, rotary dims)
SHAPES = [(16, 2, 256, 64), (6, 1, 128, 128), (4, 4, 128, 0), (5, 1, 256, 256), (24, 4, 128, 16), (7, 1, 256, 32)]
DTYPES = {torch.bfloat16: N.DTYPE_BF16, torch.float32: N.DTYPE_F32}


def shape_of(p):
    return N.FullAttnShape(p.hq, p.hk, p.d, p.rotary, p.gated)


def cache_of(p):
    return N.PagedKV(p.k, p.v, p.table)


def append(p, stream=0):
    N.full_attn_append_paged(p.weights, shape_of(p), cache_of(p), p.k_new, p.v_new, p.cu, p.kv_lens,
                             x_dtype=DTYPES[p.dtype], stream=stream)


def check_pages(p, want, before):
    k, v = want
    head = k.abs().amax(-1, keepdim=True)
    new = k != before[0].double()
    ok = (p.k.double() - k).abs() <= torch.where(new, H * k.abs() + 2e-6 * head, torch.zeros_like(k))
    same = torch.isnan(k) & torch.isnan(p.k)
    assert bool((ok | same).all())
    assert bool(((p.v.double() == v) | (torch.isnan(v) & torch.isnan(p.v))).all())


def prefill(p, out=None, scale=0.0, workspace=None, stream=0):
    s = shape_of(p)
    if out is None:
        out = torch.full((p.total, p.hq * p.d), 7.0, dtype=torch.bfloat16, device="cuda")
    if workspace is None:
        n = N.full_attn_prefill_paged_workspace_bytes(s, len(p.rows), p.total)
        workspace = torch.full((max(n, 16),), 255, dtype=torch.uint8, device="cuda")
    N.full_attn_prefill_paged(p.weights, s, cache_of(p), p.q, p.cu, p.kv_lens, out, workspace, x_dtype=DTYPES[p.dtype],
                              scale=scale, stream=stream)
    return out


def check_prefill(p, out, scale=None):
    ref, mass, reach = p.attention(scale)
    n = sum(p.rows)
    got = out.double().view(p.total, p.hq, p.d)
    tol = H * ref.abs() + (H + 2 * H * reach) * mass + 1e-30
    bad = ~((got - ref).abs() <= tol)[:n]
    assert not bool(bad.any()), (int(bad.sum()), torch.nonzero(bad)[:4].tolist())
    assert float((got - ref)[:n].norm()) <= 3 ** 0.5 * H / 3 ** 0.5 * float(ref[:n].norm()) + 1e-30
    assert bool((got[n:] == 7.0).all()), "rows behind the last sequence are left as they were"


def step(p, out_dtype, fresh=True, scale=0.0, workspace=None, out=None, stream=0):
    s = shape_of(p)
    if out is None:
        out = torch.full((len(p.rows), p.hq * p.d), 7.0, dtype=out_dtype, device="cuda")
    if workspace is None:
        n = N.full_attn_step_paged_workspace_bytes(s, len(p.rows))
        workspace = torch.full((n,), 255, dtype=torch.uint8, device="cuda")
    N.full_attn_step_paged(p.weights, s, cache_of(p), p.kv_lens, p.q, p.k_new if fresh else None,
                           p.v_new if fresh else None, out, workspace, x_dtype=DTYPES[p.dtype],
                           out_dtype=DTYPES[out_dtype], scale=scale, stream=stream)
    return out


def check_step(p, out, scale=None):
    ref, mass, reach = p.attention(scale)
    got = out.double().view(len(p.rows), p.hq, p.d)
    if out.dtype == torch.float32:
        tol = 2e-5 * mass.amax(-1, keepdim=True) + 1e-30
    else:
        tol = H * ref.abs() + 2.0 ** -16 * (1 + 2 * reach) * mass.amax(-1, keepdim=True) + 2e-5 * mass.amax() + 1e-30
    bad = ~((got - ref).abs() <= tol)
    assert not bool(bad.any()), (int(bad.sum()), torch.nonzero(bad)[:4].tolist(), float((got - ref).abs().max()))


# ---- append

@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("page,order", [(16, "rows"), (48, "heads"), (1, "rows")])
def test_append(shape, page, order, dtype):
    hq, hk, d, rotary = shape
    p = Packed([1, 0, 37, 64, 130, 5], [0, 3, 100, 0, 1, 31000], page, hq, hk, d, rotary, dtype, order,
               fused=order == "heads", seed=3, spare_rows=9)
    before, want = (p.k.clone(), p.v.clone()), p.append()
    append(p)
    check_pages(p, want, before)


def test_append_many_rows_and_no_norm():
    p = Packed([1700] + [3] * 40 + [0, 9000], [5] * 43, 64, 2, 2, 256, 64, norm=False, seed=4)
    before, want = (p.k.clone(), p.v.clone()), p.append()
    append(p)
    check_pages(p, want, before)


def test_append_skips_what_has_no_place():
    """Rows before position 0, past the table, in pages out of range, and behind the last sequence."""
    p = Packed([4, 6, 8], [-2, 10, 40], 16, 2, 2, 128, 64, seed=5, spare_rows=5)
    table = p.table.clone()
    before = p.k.clone(), p.v.clone()
    k, v = p.append()
    p.table[1, 0] = p.k.shape[0]         # sequence 1: no page holds its positions 0..15 any more
    p.table[2, 2] = -7                   # sequence 2: nor its 32..47
    p.table = p.table[:, :3].clone()     # and the table ends at 48
    page, slot = table[1, 0].long(), slice(None)
    k[page, slot], v[page, slot] = before[0][page, slot].double(), before[1][page, slot].double()
    page = table[2, 2].long()
    k[page], v[page] = before[0][page].double(), before[1][page].double()
    p.kv_lens[2] = 56                    # its last 8 rows would be at 48..55
    append(p)
    check_pages(p, (k, v), before)


# ---- decode step

@pytest.mark.parametrize("dtype,out_dtype", [(torch.bfloat16, torch.bfloat16), (torch.float32, torch.float32),
                                             (torch.bfloat16, torch.float32)])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("page,order", [(16, "rows"), (48, "heads"), (7, "rows")])
def test_step(shape, page, order, dtype, out_dtype):
    hq, hk, d, rotary = shape
    past = [0, 1, 15, 16, 62, 63, 64, 65, 300, 1023, 5000]
    p = Packed([1] * len(past), past, page, hq, hk, d, rotary, dtype, order, fused=order == "heads", seed=7,
               tail=float("nan"))
    before, want = (p.k.clone(), p.v.clone()), p.append()
    out = step(p, out_dtype)
    check_pages(p, want, before)
    check_step(p, out)


def test_step_of_appended_tokens_and_scale():
    p = Packed([1] * 3, [700, 0, 64], 16, 16, 2, 256, 64, seed=8, gated=False)
    append(p)
    check_step(p, step(p, torch.float32, fresh=False, scale=0.11), 0.11)


def test_step_one_long_sequence_many_pieces():
    p = Packed([1], [40000], 64, 16, 2, 256, 64, seed=9, tail=float("inf"))
    out = step(p, torch.float32)
    check_step(p, out)
    again = step(p, torch.float32)
    assert torch.equal(out, again), "no atomics: the same bits every time"


@pytest.mark.parametrize("batch", [129, 700])
def test_step_many_sequences(batch):
    """More sequences than threads, most of them short, some empty."""
    past = [(i * 37) % 150 for i in range(batch)]
    p = Packed([1] * batch, past, 16, 4, 1, 128, 64, seed=10)
    p.kv_lens[::5] = 0
    before = p.k.clone(), p.v.clone()
    out = step(p, torch.float32)
    none = torch.zeros(batch, dtype=torch.bool)
    none[::5] = True
    assert bool((out[none] == 0).all())
    for b in range(0, batch, 5):   # an empty sequence appends nothing
        page = p.table[b, past[b] // 16].long()
        assert torch.equal(p.k[page, past[b] % 16], before[0][page, past[b] % 16])
    p.rows = [0 if n else 1 for n in none.tolist()]
    keep = out.clone()
    p.lens = [0 if n else v + 1 for n, v in zip(none.tolist(), past)]
    ref, mass, _ = p.attention()
    got = keep.double().view(batch, 4, 128)
    # rows of the statement count packed rows: here one row a sequence, empty ones too
    for b in range(batch):
        if not none[b]:
            p1 = ref_one(p, b)
            assert float((got[b] - p1[0]).abs().max()) <= 2e-5 * float(p1[1].max())


def ref_one(p, b):
    """Sequence b's row on its own."""
    import copy
    q = copy.copy(p)
    q.rows, q.lens = [1], [p.lens[b]]
    q.cu = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    q.total, q.table, q.q = 1, p.table[b:b + 1], p.q[b:b + 1]
    out, mass, _ = q.attention()
    return out[0], mass[0]


def test_step_missing_pages_and_bad_lengths():
    p = Packed([1] * 5, [200, 200, 64, 30, 90], 16, 8, 1, 256, 64, torch.float32, seed=11, tail=float("nan"))
    append(p)
    p.table[0, 3] = -1                       # positions 48..63 are gone
    p.table[1, :12] = p.k.shape[0] + 5       # all but 192..200
    p.table[2, :] = -1                       # all of them: zeros
    p.kv_lens[3] = -4
    p.kv_lens[4] = p.table.shape[1] * 16 + 1
    k = p.k.clone()
    out = step(p, torch.float32, fresh=False)
    assert bool((out[2:] == 0).all())
    for b in (0, 1):
        ref, mass = ref_one(p, b)
        assert float((out[b].double().view(8, 256) - ref).abs().max()) <= 2e-5 * float(mass.max())
    out = step(p, torch.float32)   # the new token of sequence 2 has no page: nothing is written
    assert bool((out[2:] == 0).all())
    assert torch.equal(torch.nan_to_num(p.k), torch.nan_to_num(k))


def test_step_offsets_past_32_bits():
    """Pages whose element offsets exceed 2^31 (a cache of 4.4 GB a side)."""
    p = Packed([1], [900], 64, 16, 2, 256, 64, seed=12)
    pages = (1 << 31) // (64 * 512) + 40
    k = torch.empty(pages, 64, 2, 256, dtype=torch.bfloat16, device="cuda")
    v = torch.empty_like(k)
    table = pages - 1 - torch.arange(p.table.shape[1], dtype=torch.int32, device="cuda")[None]
    old, slots = p.table[0, :15].long(), table[0, :15].long()
    k[slots], v[slots] = p.k[old], p.v[old]
    p.k, p.v, p.table = k, v, table.contiguous()
    append(p)
    check_step(p, step(p, torch.float32, fresh=False))
    n = Packed([70], [0], 64, 16, 2, 256, 64, seed=13)
    n.k, n.v, n.table = k, v, p.table
    append(n)
    check_prefill(n, prefill(n))


# ---- prompts

@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("page,order", [(16, "rows"), (48, "heads"), (7, "rows"), (64, "heads")])
def test_prefill(shape, page, order, dtype):
    hq, hk, d, rotary = shape
    rows, past = [1, 0, 37, 64, 200, 129, 17], [0, 5, 0, 64, 0, 301, 1000]
    p = Packed(rows, past, page, hq, hk, d, rotary, dtype, order, fused=order == "heads", seed=21, spare_rows=3,
               tail=float("nan"))
    append(p)
    check_prefill(p, prefill(p))


@pytest.mark.parametrize("rows", [1, 2, 15, 16, 17, 127, 128, 129, 1000])
def test_prefill_one_prompt(rows):
    p = Packed([rows], [0], 16, 16, 2, 256, 64, seed=rows, tail=float("inf"))
    append(p)
    check_prefill(p, prefill(p))


@pytest.mark.parametrize("batch", [32, 33, 400])
@pytest.mark.parametrize("shape", [(6, 1, 128, 64), (4, 2, 256, 64)])
def test_prefill_many_sequences(shape, batch):
    """Units in the order of their lengths, over sequences of all kinds: empty ones, ones of a few
    rows behind long prefixes, several units of one length and of none (rows before position 0)."""
    hq, hk, d, rotary = shape
    rows = [(7 * i * i + 3 * i) % 23 if i % 5 else 0 if i % 2 else 60 + i % 70 for i in range(batch)]
    past = [(i * 37) % 300 if i % 3 else -(i % 11) if i % 4 else 0 for i in range(batch)]
    past = [max(x, -r) if r else max(x, 0) for x, r in zip(past, rows)]
    p = Packed(rows, past, 16, hq, hk, d, rotary, seed=26, spare_rows=2, tail=float("nan"))
    append(p)
    check_prefill(p, prefill(p))


def test_prefill_long_context_few_rows():
    p = Packed([3, 40], [20000, 9000], 64, 16, 2, 256, 64, seed=22, tail=float("nan"))
    append(p)
    out = prefill(p)
    check_prefill(p, out)
    assert torch.equal(out, prefill(p))


def test_prefill_no_gate_scale_no_norm():
    p = Packed([100, 77], [0, 10], 32, 8, 2, 128, 64, seed=23, gated=False, norm=False)
    append(p)
    check_prefill(p, prefill(p, scale=0.05), 0.05)


def test_prefill_rows_that_see_nothing():
    """Rows before position 0, a sequence without pages, and one with a hole."""
    p = Packed([20, 70, 90], [-8, 0, 100], 16, 16, 2, 256, 64, seed=24, tail=float("nan"))
    append(p)
    p.table[1, :] = -1
    p.table[2, 3:6] = p.k.shape[0]
    out = prefill(p)
    got = out.double().view(p.total, 16, 256)
    assert bool((got[:8] == 0).all()), "positions -8..-1"
    assert bool((got[20:90] == 0).all()), "no pages"
    sub = Packed([12, 0, 90], [0, 0, 100], 16, 16, 2, 256, 64, seed=24)
    sub.k, sub.v, sub.table, sub.weights = p.k, p.v, p.table, p.weights
    sub.q = torch.cat([p.q[8:20], p.q[90:180]])
    ref, mass, reach = sub.attention()
    mine = torch.cat([got[8:20], got[90:180]])
    assert bool(((mine - ref).abs() <= H * ref.abs() + (H + 2 * H * reach) * mass + 1e-30).all())


def test_prefill_large_scores():
    """Scores far apart: the running maximum moves a long way between tiles."""
    p = Packed([300], [0], 16, 4, 1, 128, 64, torch.float32, seed=25, norm=False)
    p.q[:, ::2] *= 6
    append(p)
    out = prefill(p)
    ref, mass, reach = p.attention()
    got = out.double().view(300, 4, 128)
    # scores of tens: a score off by 2^-8 reach moves weights by exp of that
    tol = H * ref.abs() + (H + torch.expm1(2 * H * reach)) * mass
    assert bool(((got - ref).abs() <= tol + 1e-30).all())


# ---- as a program uses them

def test_prompt_then_decode_in_a_graph():
    """Two prompts appended and attended, then three decode steps replayed from one captured graph of
    append-and-step on a side stream, each against the statement; the graph of one step serves all."""
    steps = 3
    p = Packed([45, 130], [0, 0], 16, 16, 2, 256, 64, seed=31)
    extra = Packed([1, 1], [45 + steps, 130 + steps], 16, 16, 2, 256, 64, seed=32)
    p.table, p.k, p.v = extra.table, extra.k, extra.v
    append(p)
    check_prefill(p, prefill(p))
    d = Packed([1, 1], [45, 130], 16, 16, 2, 256, 64, torch.float32, seed=33)
    d.table, d.k, d.v, d.weights = p.table, p.k, p.v, p.weights
    shape, cache = shape_of(d), cache_of(d)
    ws = torch.empty(N.full_attn_step_paged_workspace_bytes(shape, 2), dtype=torch.uint8, device="cuda")
    out = torch.empty(2, 16 * 256, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    lens0 = d.kv_lens.clone()
    with torch.cuda.stream(side):
        step(d, torch.float32, workspace=ws, out=out, stream=side.cuda_stream)
        side.synchronize()
        with torch.cuda.graph(graph, stream=side):
            step(d, torch.float32, workspace=ws, out=out, stream=side.cuda_stream)
    torch.cuda.synchronize()
    for i in range(steps):
        d.kv_lens.copy_(lens0 + i)
        d.lens = [46 + i, 131 + i]
        for t in (d.q, d.k_new, d.v_new):
            t.normal_()
        before, want = (d.k.clone(), d.v.clone()), d.append()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        check_pages(d, want, before)
        check_step(d, out)


def test_step_agrees_with_the_dense_step():
    """The same tokens through nmoe_full_attn_step_batched (dense bf16 cache)."""
    B, cap = 3, 128
    past = [0, 63, 100]
    p = Packed([1] * B, past, 16, 16, 2, 256, 64, torch.float32, seed=41)
    kc, vc = (torch.zeros(B, cap, 2, 256, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    for b in range(B):
        page, slot = p.places(b)
        kc[b, :past[b]], vc[b, :past[b]] = p.k[page, slot][:past[b]], p.v[page, slot][:past[b]]
    ws = torch.zeros(N.full_attn_batched_workspace_bytes(B) // 4, dtype=torch.int32, device="cuda")
    dense = torch.zeros(B, 16 * 256, device="cuda")
    pos = torch.tensor(past, dtype=torch.int32, device="cuda")
    N.full_attn_step_batched(p.weights, p.q, p.k_new, p.v_new, kc, vc, pos, cap, dense, ws)
    out = step(p, torch.float32)
    # the new key may round to the neighbouring bf16 value (2^-7 of one of up to 101 positions)
    assert float((out - dense).abs().max()) <= 1e-3 * float(dense.abs().max())


def test_two_streams_with_workspaces_of_their_own():
    a = Packed([1] * 4, [3000, 10, 500, 64], 16, 16, 2, 256, 64, torch.float32, seed=51)
    b = Packed([200, 33], [0, 50], 16, 16, 2, 256, 64, seed=52)
    append(b)
    size = lambda n: torch.full((max(n, 16),), 255, dtype=torch.uint8, device="cuda")  # noqa: E731
    w1 = size(N.full_attn_step_paged_workspace_bytes(shape_of(a), 4))
    w2 = size(N.full_attn_prefill_paged_workspace_bytes(shape_of(b), 2, b.total))
    # memory that lives until both streams are done (the helpers' own buffers belong to the default stream)
    x = [torch.full((4, 4096), 7.0, device="cuda") for _ in range(5)]
    y = [torch.full((b.total, 4096), 7.0, dtype=torch.bfloat16, device="cuda") for _ in range(5)]
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    outs = [(step(a, torch.float32, workspace=w1, out=x[i], stream=s1.cuda_stream),
             prefill(b, workspace=w2, out=y[i], stream=s2.cuda_stream)) for i in range(5)]
    torch.cuda.synchronize()
    for x, y in outs:
        check_step(a, x)
        check_prefill(b, y)


def test_no_rows():
    p = Packed([0, 0], [5, 0], 16, 16, 2, 256, 64, seed=61)
    before = p.k.clone()
    append(p)
    prefill(p)
    assert torch.equal(before, p.k)
    empty = Packed([1], [0], 16, 16, 2, 256, 64, seed=62)
    s = shape_of(empty)
    N.full_attn_step_paged(empty.weights, s, cache_of(empty), empty.kv_lens[:0], empty.q[:0], None, None,
                           torch.empty(0, 4096, dtype=torch.bfloat16, device="cuda"),
                           torch.empty(16, dtype=torch.uint8, device="cuda"), x_dtype=N.DTYPE_BF16,
                           out_dtype=N.DTYPE_BF16)
