"""Paged full-attention calls one after the other on one workspace: what a call leaves running when
its outputs are there would be found by the next one."""
import pytest
import torch

import nmoe_b200 as N
from operators_ref import Packed
from test_paged_attn_gpu import append, check_pages, check_prefill, prefill, shape_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,cu", [([4000, 3000, 77], None), ([0, 0], [0, 0, 0]), ([4000], [0, 0])])
def test_prefill_behind_one_in_which_no_row_sees_anything(rows, cu):
    """All rows before position 0, or none of a sequence (a batch padded for a captured graph): no unit needs the
    prepared queries, and the launch that prepares them still writes the workspace that the next call takes."""
    blind = Packed(rows, [-r for r in rows], 16, 16, 2, 256, 64, seed=71, spare_rows=6000)
    if cu is not None:
        blind.cu = torch.tensor(cu, dtype=torch.int32, device="cuda")
    p = Packed([130, 45], [0, 7], 16, 16, 2, 256, 64, seed=72)
    append(p)
    size = N.full_attn_prefill_paged_workspace_bytes(shape_of(blind), len(rows), blind.total)
    ws = torch.full((size,), 255, dtype=torch.uint8, device="cuda")
    outs = [torch.full((p.total, 4096), 7.0, dtype=torch.bfloat16, device="cuda") for _ in range(8)]
    none = torch.full((blind.total, 4096), 7.0, dtype=torch.bfloat16, device="cuda")
    torch.cuda.synchronize()
    for out in outs:
        prefill(blind, out=none, workspace=ws)
        prefill(p, out=out, workspace=ws)
    torch.cuda.synchronize()
    n = sum(rows) if cu is None else 0
    assert bool((none[:n] == 0).all()) and bool((none[n:] == 7.0).all())
    for out in outs:
        assert torch.equal(out, outs[0])
    check_prefill(p, outs[0])


@pytest.mark.parametrize("heads", [(16, 2, 256, 64), (6, 1, 128, 128)])
def test_rows_in_front_of_the_first_sequence(heads):
    """cu_rows need not begin at zero: what lies in front belongs to no sequence."""
    p = Packed([130, 0, 45], [20, 3, 0], 16, *heads, seed=73, tail=float("nan"))
    before, want = (p.k.clone(), p.v.clone()), p.append()
    q, out = p.q.clone(), torch.full((p.total + 9, p.hq * p.d), 7.0, dtype=torch.bfloat16, device="cuda")
    front = lambda t: torch.cat([torch.full((9, t.shape[1]), float("nan"), dtype=t.dtype, device="cuda"), t])  # noqa: E731
    p.q, p.k_new, p.v_new = front(p.q), front(p.k_new), front(p.v_new)
    p.cu += 9
    p.total += 9
    append(p)
    check_pages(p, want, before)
    prefill(p, out=out)
    assert bool((out[:9] == 7.0).all())
    p.q, p.cu, p.total = q, p.cu - 9, p.total - 9
    check_prefill(p, out[9:])
