"""nmoe_linear_attn_prefill where magnitudes change on the way, against the 64-bit statement; the
tolerances are those of test_linear_attn_prefill_gpu."""
import pytest
import torch

import nmoe_b200 as N  # noqa: F401  (the extension has to be there)
from operators_ref import gdn
from test_linear_attn_prefill_gpu import TOL, Prompt

pytestmark = pytest.mark.gpu


def statement(p):
    conv, delta = p.conv.double().clone(), p.delta.double().clone()
    return gdn(p.w, p.hk, p.hv, p.cu_host, p.qkv, p.z, p.alpha, p.beta, conv, delta), conv, delta


@pytest.mark.parametrize("dims,rows", [(8, 640), (128, 1500)])
@pytest.mark.parametrize("size", [1.0, 1e5, 1e7])
def test_a_large_start_that_the_rule_erases(dims, rows, size):
    """16 large values, then ordinary ones, without decay: keys along the first `dims` axes in turn and
    a step of 0.999, so that a visit to a key leaves a thousandth of what its column of the state held.

    What a visit rounds, 2^-24 of the column or 2^-32 of the largest value of a chunk and of the two
    before it, is erased by the next visits too. A large column is visited 8 times or more before the rows that
    are compared: 1e7 * 1e-3^8 is nothing. So their error is that of ordinary values, whatever the start was."""
    p = Prompt([rows], 1, 1, torch.float32, seed=21, fresh=True)
    p.w["conv_w"].zero_()
    p.w["conv_w"][:, 3] = 1.0
    p.w["A_log"].zero_(), p.w["dt_bias"].zero_()
    p.qkv[:, 128:256] = 0
    t = torch.arange(rows, device="cuda")
    p.qkv[t, 128 + t % dims] = 10.0
    p.qkv[:16, 256:] = p.qkv[:16, 256:].abs() * size
    p.alpha[:], p.beta[:] = -12.0, 7.0
    out, conv, delta = p.run()
    ref, c64, d64 = statement(p)
    assert torch.equal(conv.double(), c64)
    assert float((delta.double() - d64).abs().max()) <= TOL * float(d64.abs().max())
    late = slice(rows * 3 // 4, rows)
    assert float((out.double() - ref)[late].abs().max()) <= TOL * float(ref[late].abs().max())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_decays_that_forget_everything(dtype):
    """A gate so large, up to infinity, that nothing of the state is left: what follows in the same chunk goes on
    from there, with the small decays between its own tokens. And gates of -inf: no decay at all."""
    p = Prompt([150, 40], 1, 2, dtype, seed=22)
    for row, size in ((5, 1e4), (20, 1e12), (37, 1e30), (64, 3e38), (80, float("inf")), (81, float("inf")), (127, 1e9), (160, 2e20)):
        p.alpha[row] = size
    p.alpha[100, 1] = float("inf")
    p.alpha[30:34] = p.alpha[90] = float("-inf")
    p.check(*p.run())


@pytest.mark.parametrize("heads,rows,dtype,out_dtype", [
    ((16, 32), [6000], torch.bfloat16, torch.bfloat16), ((4, 4), [5000, 6100], torch.float32, torch.bfloat16),
    ((2, 6), [5900, 3], torch.bfloat16, torch.float32)])
def test_parts_of_several_key_heads(heads, rows, dtype, out_dtype):
    """Three parts or more of a prompt: the norm of an earlier part runs in rows of the grid between those of the key
    heads, whatever their number."""
    p = Prompt(rows, *heads, dtype, seed=23, spare=2)
    p.check(*p.run(out_dtype))


@pytest.mark.parametrize("heads", [(1, 3), (2, 6), (1, 5)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_odd_numbers_of_value_heads_a_key_head(heads, dtype):
    p = Prompt([1, 70, 0, 130, 64], *heads, dtype, seed=24, spare=1)
    p.check(*p.run())


@pytest.mark.parametrize("scale", [1e9, 1e13])
def test_large_values(scale):
    p = Prompt([150, 0, 70], 1, 2, torch.float32, seed=25, scale=scale)
    p.conv *= scale
    p.check(*p.run())


@pytest.mark.parametrize("rows", [[100, 130, 70], [100] * 20 + [130] + [50] * 20, [9000, 9100, 9003]])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_what_is_not_finite_stays_in_its_sequence(rows, bad):
    """Every operand of one row set to NaN or an infinity, each in a sequence of its own kind: the other sequences give
    the same bits, and so do the chunks before it."""
    at = rows.index(max(rows)) if len(rows) > 3 else 1
    for which in ("qkv", "z", "alpha", "beta", "state"):
        p = Prompt(rows, 1, 2, torch.float32, seed=26)
        clean = p.run()
        first = p.cu_host[at] + 70
        if which == "state":
            p.delta[at, 1, 3, 5] = bad
            p.conv[at, 1, 7] = bad
            first = p.cu_host[at]
        else:
            getattr(p, which)[first] = bad
            if which == "qkv":
                p.qkv[first, 1:] = 1.0   # one channel of a query
        out, conv, delta = p.run()
        end = p.cu_host[at + 1]
        before = p.cu_host[at] + (first - p.cu_host[at]) // 64 * 64
        assert torch.equal(out[:before], clean[0][:before]) and torch.equal(out[end:], clean[0][end:]), which
        others = [b for b in range(len(rows)) if b != at]
        assert torch.equal(conv[others], clean[1][others]) and torch.equal(delta[others], clean[2][others]), which


def test_rows_in_front_of_the_first_sequence():
    """cu_rows need not begin at zero: what lies in front belongs to no sequence."""
    p = Prompt([11, 70, 5], 1, 2, torch.float32, seed=27, spare=2)
    p.cu_host = [c + 7 for c in [0, 60, 60, 79]]
    p.cu = torch.tensor(p.cu_host, dtype=torch.int32, device="cuda")
    out, conv, delta = p.run()
    assert bool((out[:7] == 7.0).all())
    out[:7] = 0   # the statement's value for rows that it does not compute
    p.check(out, conv, delta)
