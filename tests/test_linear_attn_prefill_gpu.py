"""nmoe_linear_attn_prefill on the GPU against the token-by-token 64-bit statement
(operators_ref.gdn): conv state bit-exact (copies), recurrent state and fp32 output within 2e-5 of
the largest magnitude (the tolerance of the single-token step: fp32 sums in another order), a bf16
output within half a bf16 step, 2^-8 of the value, beside that."""
import pytest
import torch

import nmoe_b200 as N
from operators_ref import gdn

pytestmark = pytest.mark.gpu
TOL, H = 2e-5, 2.0 ** -8


class Prompt:
    def __init__(self, rows, hk=2, hv=4, dtype=torch.float32, seed=0, fresh=False, spare=0, fused=False, scale=1.0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        rnd = lambda *s, std=1.0: torch.randn(s, generator=g, device="cuda") * std  # noqa: E731
        self.rows, self.hk, self.hv, self.dtype = rows, hk, hv, dtype
        self.cu_host = [sum(rows[:i]) for i in range(len(rows) + 1)]
        self.cu = torch.tensor(self.cu_host, dtype=torch.int32, device="cuda")
        self.total, ch = sum(rows) + spare, (2 * hk + hv) * 128
        wide = [ch, hv * 128, hv, hv]
        if fused:   # one projection's rows, padded to 16-byte rows
            pad = -sum(wide) % 8
            x = (rnd(self.total, sum(wide) + pad) * scale).to(dtype)
            self.qkv, self.z, self.alpha, self.beta, _ = x.split(wide + [pad], 1)
        else:
            self.qkv, self.z, self.alpha, self.beta = (rnd(self.total, n).to(dtype) for n in wide)
            self.qkv = (self.qkv * scale).to(dtype)
        self.w = {"conv_w": rnd(ch, 4, std=0.3).bfloat16(), "A_log": rnd(hv, std=0.5),
                  "dt_bias": rnd(hv, std=0.5).bfloat16(), "norm_w": (rnd(128, std=0.1) + 1).bfloat16()}
        n = len(rows)
        self.conv = rnd(n, 3, ch) * (0.0 if fresh else 1.0)
        self.delta = rnd(n, hv, 128, 128, std=0.05) * (0.0 if fresh else 1.0)
        self.fresh = fresh

    def run(self, out_dtype=torch.float32, in_place=False, null_in=False, workspace=None, stream=0):
        s = N.LinearAttnShape(self.hk, self.hv)
        if workspace is None:
            n = N.linear_attn_prefill_workspace_bytes(s, len(self.rows), self.total)
            workspace = torch.full((max(n, 16),), 255, dtype=torch.uint8, device="cuda")
        out = torch.full((self.total, self.hv * 128), 7.0, dtype=out_dtype, device="cuda")
        conv = self.conv.clone() if in_place else torch.full_like(self.conv, 7.0)
        delta = self.delta.clone() if in_place else torch.full_like(self.delta, 7.0)
        code = {torch.bfloat16: N.DTYPE_BF16, torch.float32: N.DTYPE_F32}
        cin, din = (conv, delta) if in_place else (None, None) if null_in else (self.conv, self.delta)
        N.linear_attn_prefill(self.w, s, self.qkv, self.z, self.alpha, self.beta, self.cu, cin, din, conv, delta, out,
                              workspace, x_dtype=code[self.dtype], out_dtype=code[out_dtype], stream=stream)
        return out, conv, delta

    def check(self, out, conv, delta):
        c64, d64 = self.conv.double().clone(), self.delta.double().clone()
        ref = gdn(self.w, self.hk, self.hv, self.cu_host, self.qkv, self.z, self.alpha, self.beta, c64, d64)
        n = self.cu_host[-1]
        assert torch.equal(conv.double(), c64)
        assert float((delta.double() - d64).abs().max()) <= TOL * max(float(d64.abs().max()), 1e-6)
        if n:
            err = (out.double() - ref)[:n].abs()
            tol = TOL * float(ref.abs().max()) + (H * ref[:n].abs() if out.dtype == torch.bfloat16 else 0)
            assert bool((err <= tol).all()), float(err.max())
        assert bool((out[n:] == 7.0).all()), "rows behind the last sequence are left as they were"


@pytest.mark.parametrize("dtype,out_dtype", [(torch.bfloat16, torch.bfloat16), (torch.float32, torch.float32),
                                             (torch.bfloat16, torch.float32), (torch.float32, torch.bfloat16)])
@pytest.mark.parametrize("heads", [(2, 4), (1, 1), (3, 3), (1, 4)])
def test_packed(heads, dtype, out_dtype):
    p = Prompt([1, 0, 2, 3, 64, 65, 130, 17], *heads, dtype, seed=1, spare=5, fused=heads == (2, 4))
    p.check(*p.run(out_dtype))


@pytest.mark.parametrize("rows", [1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 128, 129, 200])
def test_lengths(rows):
    p = Prompt([rows], 1, 2, torch.float32, seed=rows)
    p.check(*p.run())


@pytest.mark.parametrize("count", [32, 33, 300])
def test_many_sequences(count):
    p = Prompt([(11 * i * i + 5 * i) % 7 if i % 9 else 60 + i % 70 for i in range(count)], 1, 2, torch.bfloat16, seed=17, spare=1)
    p.check(*p.run())


def test_full_geometry_and_new_sequences():
    p = Prompt([100, 33], 16, 32, torch.bfloat16, seed=3, fresh=True)
    p.check(*p.run(torch.bfloat16, null_in=True))


def test_long_prompt():
    p = Prompt([1500], 1, 2, torch.float32, seed=4)
    p.check(*p.run())


def test_states_in_place_and_the_same_bits_twice():
    p = Prompt([70, 0, 129, 1], 2, 4, torch.float32, seed=5)
    a, b = p.run(in_place=True), p.run()
    for x, y in zip(a, b):
        assert torch.equal(x, y)
    p.check(*a)


@pytest.mark.parametrize("scale", [1e-4, 300.0])
def test_value_ranges(scale):
    """Inputs far from one: the conv output, and with it the state, scales with them."""
    p = Prompt([150, 20], 1, 2, torch.float32, seed=6, scale=scale)
    p.conv *= scale
    p.check(*p.run())


def test_slow_and_fast_decay_and_alike_keys():
    """Keys that are nearly the same at every token, decay near one, beta near one: the triangular
    system of a chunk at its worst."""
    p = Prompt([140], 1, 2, torch.float32, seed=7)
    p.qkv[:, 128:256] = p.qkv[:1, 128:256] + 0.02 * p.qkv[:, 128:256]
    p.alpha[:, 0], p.alpha[:, 1] = -8.0, 6.0
    p.beta[:] = 6.0
    p.check(*p.run())


def test_a_large_state_that_decays_with_nothing_new():
    """A state of 1e6 that loses 23 decades a chunk while every value is zero.

    Operands are held to an absolute error too. Scaled so that 2^12 <= B 2^-e < 2^13, B the bound
    sqrt(128) max|S| on them, an element is off by half of fp16's least step, 2^-25 2^e; with e one
    larger for R that is 2^-36 B at most. An output element before its norm is a sum over 64 tokens of
    R's elements, each times a product of q, contractions and k: at most |q| = 128^-1/2. So it is
    off by 64 * 128^-1/2 * 2^-36 * 128^1/2 max|S| = 2^-30 max|S|, and by less again through S itself:
    2^-29 max|S|. The norm divides by the row's root mean square r and passes on at most twice
    that; r follows from the 64-bit output y / (w silu(z)), whose mean square is r^2 / (r^2 + 1e-6)."""
    p = Prompt([200], 1, 1, torch.float32, seed=16)
    p.qkv[:, 256:] = 0
    p.conv[:, :, 256:] = 0
    p.delta *= 2e7
    p.w["A_log"][:], p.w["dt_bias"][:] = 0.0, 0.0
    p.alpha[:] = 0.24
    out, conv, delta = p.run()
    c64, d64 = p.conv.double().clone(), p.delta.double().clone()
    ref = gdn(p.w, 1, 1, p.cu_host, p.qkv, p.z, p.alpha, p.beta, c64, d64)
    gate = (p.w["norm_w"].double() * torch.nn.functional.silu(p.z.double())).abs()
    m = (ref / gate).pow(2).mean(1, keepdim=True)
    r = (1e-6 * m / (1 - m) + 1e-6).sqrt()
    tol = TOL * float(ref.abs().max()) + 2 * 2.0 ** -29 * float(p.delta.abs().max()) / r * gate
    assert bool(((out.double() - ref).abs() <= tol).all())
    assert float((delta.double() - d64).abs().max()) <= 1e-20


def test_zero_keys():
    p = Prompt([80], 1, 1, torch.float32, seed=8, fresh=True)
    p.qkv[20:50] = 0
    p.check(*p.run())


def test_chunks_of_a_prompt_then_single_steps():
    """A prompt in two chunks, then nmoe_linear_attn_step_batched from the states they leave."""
    w, steps = 16, 3
    whole = Prompt([90, 41], 16, 32, torch.float32, seed=9, fresh=True)
    conv, delta = whole.conv.double().clone(), whole.delta.double().clone()
    cut = [50, 41]

    def part(lo, hi):
        p = Prompt([h - l for l, h in zip(lo, hi)], 16, 32, torch.float32, seed=0)
        rows = torch.cat([torch.arange(whole.cu_host[b] + l, whole.cu_host[b] + h) for b, (l, h) in enumerate(zip(lo, hi))])
        p.w, p.qkv, p.z, p.alpha, p.beta = whole.w, *(t[rows.cuda()].contiguous() for t in (whole.qkv, whole.z, whole.alpha, whole.beta))
        return p

    a = part([0, 0], cut)
    a.conv.zero_(), a.delta.zero_()
    out1, a_conv, a_delta = a.run(null_in=True)
    b = part(cut, [90 - steps, 41])
    b.conv, b.delta = a_conv, a_delta
    out2, c, d = b.run(in_place=True)
    ref = gdn(whole.w, 16, 32, [0, 90], whole.qkv, whole.z, whole.alpha, whole.beta, conv[:1], delta[:1])
    got = torch.cat([out1[:50], out2[:40 - steps]])
    tol = TOL * float(ref.abs().max())
    assert float((got.double() - ref[:90 - steps]).abs().max()) <= tol
    # the last tokens of sequence 0 one at a time, from the states the prompt left
    c1, d1 = c[:1].contiguous(), d[:1].contiguous()
    for r in range(90 - steps, 90):
        o = torch.empty(1, 4096, device="cuda")
        N.linear_attn_step_batched(whole.w, whole.qkv[r:r + 1], whole.z[r:r + 1], whole.alpha[r:r + 1],
                                   whole.beta[r:r + 1], c1, d1, o)
        assert float((o[0].double() - ref[r]).abs().max()) <= tol
    assert float((d1.double() - delta[:1]).abs().max()) <= TOL * float(delta.abs().max())


def test_in_a_graph_on_a_side_stream():
    p = Prompt([77, 5], 2, 4, torch.float32, seed=11)
    s = N.LinearAttnShape(2, 4)
    ws = torch.empty(max(16, N.linear_attn_prefill_workspace_bytes(s, 2, p.total)), dtype=torch.uint8, device="cuda")
    out, conv, delta = torch.empty(p.total, 512, device="cuda"), torch.empty_like(p.conv), torch.empty_like(p.delta)
    call = lambda st: N.linear_attn_prefill(p.w, s, p.qkv, p.z, p.alpha, p.beta, p.cu, p.conv, p.delta, conv, delta, out, ws,  # noqa: E731
                                            x_dtype=N.DTYPE_F32, out_dtype=N.DTYPE_F32, stream=st)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        call(side.cuda_stream)
        side.synchronize()
        with torch.cuda.graph(graph, stream=side):
            call(side.cuda_stream)
    for rows in ([77, 5], [40, 42], [0, 82]):
        p.cu_host = [0, rows[0], 82]
        p.cu.copy_(torch.tensor(p.cu_host, dtype=torch.int32))
        p.qkv.normal_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        p.check(out, conv, delta)


def test_no_rows_keep_the_states():
    p = Prompt([0, 0], 1, 1, torch.float32, seed=12)
    out, conv, delta = p.run()
    assert torch.equal(conv, p.conv) and torch.equal(delta, p.delta)


@pytest.mark.parametrize("rows,dtype", [([9001], torch.bfloat16), ([17390, 30], torch.float32), ([5200, 0, 70, 5201], torch.float32)])
def test_prompts_prepared_in_parts(rows, dtype):
    """Long sequences that leave most of the machine idle: their chunks go in parts, each prepared while
    the scan of the part before runs, the state handed on through memory. The state in place, one
    sequence shorter than the parts are many, and the same from a captured graph, replayed twice."""
    p = Prompt(rows, 1, 2, dtype, seed=13, spare=3)
    a = p.run(in_place=True)
    p.check(*a)
    s = N.LinearAttnShape(1, 2)
    ws = torch.empty(N.linear_attn_prefill_workspace_bytes(s, len(rows), p.total), dtype=torch.uint8, device="cuda")
    out, conv, delta = torch.full_like(a[0], 7.0), torch.empty_like(p.conv), torch.empty_like(p.delta)
    code = N.DTYPE_BF16 if dtype == torch.bfloat16 else N.DTYPE_F32
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        N.linear_attn_prefill(p.w, s, p.qkv, p.z, p.alpha, p.beta, p.cu, p.conv, p.delta, conv, delta, out, ws,
                              x_dtype=code, out_dtype=N.DTYPE_F32, stream=side.cuda_stream)
    for _ in range(2):
        ws.fill_(255)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(a, (out, conv, delta)):
            assert torch.equal(x, y)


def test_two_streams_with_workspaces_of_their_own():
    """Two calls at once, one of them in parts, give what each gives alone."""
    a, b = Prompt([9001], 1, 2, torch.bfloat16, seed=14), Prompt([700, 64, 1300], 4, 8, torch.float32, seed=15)
    alone = [p.run() for p in (a, b)]
    calls = []
    for p, code in ((a, N.DTYPE_BF16), (b, N.DTYPE_F32)):
        s = N.LinearAttnShape(p.hk, p.hv)
        ws = torch.full((N.linear_attn_prefill_workspace_bytes(s, len(p.rows), p.total),), 255, dtype=torch.uint8, device="cuda")
        outs = [(torch.full((p.total, p.hv * 128), 7.0, device="cuda"), torch.empty_like(p.conv), torch.empty_like(p.delta))
                for _ in range(4)]
        calls.append((p, s, ws, outs, torch.cuda.Stream(), code))
    torch.cuda.synchronize()
    for i in range(4):
        for p, s, ws, outs, stream, code in calls:
            out, conv, delta = outs[i]
            N.linear_attn_prefill(p.w, s, p.qkv, p.z, p.alpha, p.beta, p.cu, p.conv, p.delta, conv, delta, out, ws,
                                  x_dtype=code, out_dtype=N.DTYPE_F32, stream=stream.cuda_stream)
    torch.cuda.synchronize()
    for want, (_, _, _, outs, _, _) in zip(alone, calls):
        for got in outs:
            for x, y in zip(want, got):
                assert torch.equal(x, y)
