"""The operators that take whole prompts, and single tokens over a paged key-value cache, through the
two kinds of attention layers that the library's decode step has: their cases, their plain forms and
the calls that a program makes of them.

  append   keys normalised, rotated and appended, with the values, to a paged bf16 cache
  step     one new token per sequence: append, then attention over its pages
  prefill  causal grouped-head attention of packed prompts over their pages
  gdn      the gated delta rule of a linear-attention layer over packed prompts (convolution, key and
           query norms, decay, delta rule, gated norm), states in and out

Sequences are packed: sequence b's rows are cu_rows[b] .. cu_rows[b + 1] - 1, and its cache holds
kv_lens[b] positions once they are appended, the rows being the last of them.
"""
import math
import os
import random
import sys

import torch

own = False

BF16, F32 = "bf16", "f32"
TORCH = {BF16: torch.bfloat16, F32: torch.float32}
THETA = 10000000.0   # rotation base, the decode step's
EPS = 1e-6


def _text(lengths):
    return ",".join(str(int(v)) for v in lengths)


def _lengths(text):
    return [int(v) for v in text.split(",")]


def _ragged(rng, count, total):
    """`count` lengths, some zero or one, that add up to `total`."""
    w = [0.0 if rng.random() < 0.05 else math.exp(rng.uniform(0, 4)) for _ in range(count)]
    w[rng.randrange(count)] += math.exp(3)
    got = [int(total * x / sum(w)) for x in w]
    got[max(range(count), key=lambda i: got[i])] += total - sum(got)
    return got


# ---- cases ---------------------------------------------------------------------------------------

def _attn(op, name, rows, past, page, dtype, q_heads=16, kv_heads=2, head_dim=256, rotary=64, order="rows", fused=False):
    return {"name": name, "op": op, "rows": _text(rows), "past": _text(past), "page": page, "dtype": dtype,
            "q_heads": q_heads, "kv_heads": kv_heads, "head_dim": head_dim, "rotary": rotary, "order": order,
            "fused": fused}


def _gdn(name, rows, dtype, key_heads=16, value_heads=32, fresh=True):
    return {"name": name, "op": "gdn", "rows": _text(rows), "dtype": dtype, "key_heads": key_heads,
            "value_heads": value_heads, "fresh": fresh}


def listed():
    r = random.Random(11)
    return [
        # the cache write of one decode step of 64 sequences, where the launch is what costs
        _attn("append", "append_64x1", [1] * 64, [r.randrange(0, 4096) for _ in range(64)], 16, BF16),
        # a ragged batch of prompts in fp32, head-major pages, one prompt behind a cached prefix
        _attn("append", "append_ragged_f32", [1, 900, 37, 0, 2100, 64, 994], [0, 500, 0, 9, 0, 0, 3], 64, F32,
              order="heads"),
        # the prompts of a large prefill batch, read out of one fused projection's rows
        _attn("append", "append_32768", [8192] * 4, [0] * 4, 64, BF16, fused=True),
        # batch-1 decode at a context of 4096
        _attn("step", "step_1x4096", [1], [4095], 64, BF16),
        # a ragged decode batch in fp32: one sequence new, the others up to 16384 long
        _attn("step", "step_ragged_f32", [1] * 37, [0] + [int(16384 ** r.random()) for _ in range(35)] + [16383], 16,
              F32, q_heads=32, kv_heads=4, head_dim=128, rotary=128),
        # throughput decode: 64 sequences, each at a context of 32768
        _attn("step", "step_64x32768", [1] * 64, [32767] * 64, 64, BF16, fused=True),
        # a short question: latency counts
        _attn("prefill", "prefill_37", [37], [0], 16, BF16),
        # prompts and chunks of prompts packed together, some behind a cached prefix, odd lengths
        _attn("prefill", "prefill_ragged", [513, 1, 1800, 77, 0, 3000, 605], [0, 4000, 900, 0, 12, 0, 8191], 32, BF16,
              q_heads=24, kv_heads=4, head_dim=128, rotary=64, order="heads"),
        # one long prompt
        _attn("prefill", "prefill_16384", [16384], [0], 64, BF16, fused=True),
        # a short question
        _gdn("gdn_53", [53], BF16),
        # packed prompts of odd lengths in fp32 that go on from earlier states
        _gdn("gdn_ragged_f32", [513, 1, 1800, 77, 0, 2, 1003, 64, 605], F32, fresh=False),
        # one long prompt: the recurrence is the long axis
        _gdn("gdn_16384", [16384], BF16),
    ]


def draw(rng):
    op = rng.choice(["append", "step", "prefill", "gdn"])
    dtype = rng.choice([BF16, F32])
    log = lambda lo, hi: int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))  # noqa: E731
    if op == "gdn":
        key_heads = rng.choice([2, 4, 8, 16])
        count = log(1, 12)
        total = max(count, log(16, 12000))
        return {k: v for k, v in _gdn("", _ragged(rng, count, total), dtype, key_heads,
                                      key_heads * rng.choice([1, 2]), rng.random() < 0.5).items() if k != "name"}
    head_dim = rng.choice([128, 256])
    kv_heads = rng.choice([1, 2, 3, 4])
    group = rng.choice([1, 2, 4, 5, 6, 8])
    page = rng.choice([8, 16, 32, 48, 64, 128])
    rotary = rng.choice([0, 64, 128])
    width = kv_heads * head_dim
    if op == "append":
        count = log(1, 64)
        total = max(count, log(8, 16384 * 512 // width))
        rows = _ragged(rng, count, total)
        past = [rng.choice([0, log(1, 2000)]) for _ in rows]
    elif op == "step":
        count = log(1, 48)
        longest = min(32768, max(64, 48 * 8192 * 512 // (count * width)))
        rows = [1] * count
        past = [rng.choice([0, 1, log(1, longest), log(1, longest), longest - 1]) for _ in rows]
    else:
        count = log(1, 8)
        total = max(count, log(8, 8000))
        rows = _ragged(rng, count, total)
        past = [rng.choice([0, 0, log(1, 4000)]) for _ in rows]
    c = _attn(op, "", rows, past, page, dtype, kv_heads * group, kv_heads, head_dim, rotary,
              rng.choice(["rows", "heads"]), rng.random() < 0.5)
    return {k: v for k, v in c.items() if k != "name"}


# ---- inputs --------------------------------------------------------------------------------------

def _randn(gen, shape, dtype=torch.float32, std=1.0, mean=0.0):
    return (torch.randn(shape, generator=gen, device="cuda") * std + mean).to(dtype)


def _cumulative(lengths):
    cu = [0]
    for n in lengths:
        cu.append(cu[-1] + n)
    return torch.tensor(cu, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    return _prepare_gdn(case, seed) if case["op"] == "gdn" else _prepare_attn(case, seed)


def _prepare_attn(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(1000003 * seed + 17)
    rows, past = _lengths(case["rows"]), _lengths(case["past"])
    total, seqs = sum(rows), len(rows)
    hq, hk, d, page = case["q_heads"], case["kv_heads"], case["head_dim"], case["page"]
    dtype = TORCH[case["dtype"]]
    lens = [a + b for a, b in zip(past, rows)]
    # pages in a shuffled order, a few of them free; what lies behind a sequence's end is left over
    # from earlier use
    need = [-(-n // page) for n in lens]
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    table = torch.zeros(seqs, max(1, max(need)), dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    shape = (pages, page, hk, d) if case["order"] == "rows" else (pages, hk, page, d)
    k_pages = torch.empty(shape, dtype=torch.bfloat16, device="cuda").normal_(generator=gen)
    v_pages = torch.empty(shape, dtype=torch.bfloat16, device="cuda").normal_(generator=gen)
    if case["order"] == "heads":
        k_pages, v_pages = k_pages.transpose(1, 2), v_pages.transpose(1, 2)
    # a layer's q (query | gate per head), k and v: of their own, or side by side in a fused projection's rows
    wide = [hq * 2 * d, hk * d, hk * d]
    if case["fused"]:
        q, k_new, v_new = _randn(gen, (total, sum(wide)), dtype).split(wide, dim=1)
    else:
        q, k_new, v_new = (_randn(gen, (total, w), dtype) for w in wide)
    return {"op": case["op"], "case": case, "seqs": seqs, "total": total, "rows": rows, "lens": lens,
            "cu_rows": _cumulative(rows), "kv_lens": torch.tensor(lens, dtype=torch.int32, device="cuda"),
            "table": table, "k_pages": k_pages, "v_pages": v_pages, "q": q, "k_new": k_new, "v_new": v_new,
            "q_norm": _randn(gen, (d,), torch.bfloat16, 0.1), "k_norm": _randn(gen, (d,), torch.bfloat16, 0.1),
            "kept": {}}


def _prepare_gdn(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(1000003 * seed + 29)
    rows = _lengths(case["rows"])
    total, seqs, hk, hv = sum(rows), len(rows), case["key_heads"], case["value_heads"]
    dtype = TORCH[case["dtype"]]
    ch = (2 * hk + hv) * 128
    s = {"op": "gdn", "case": case, "seqs": seqs, "total": total, "rows": rows, "cu_rows": _cumulative(rows),
         "qkv": _randn(gen, (total, ch), dtype), "z": _randn(gen, (total, hv * 128), dtype),
         "alpha": _randn(gen, (total, hv), dtype), "beta": _randn(gen, (total, hv), dtype),
         "conv_w": _randn(gen, (ch, 4), torch.bfloat16, 0.3), "A_log": _randn(gen, (hv,), std=0.5),
         "dt_bias": _randn(gen, (hv,), torch.bfloat16, 0.5), "norm_w": _randn(gen, (128,), torch.bfloat16, 0.1, 1.0),
         "kept": {}}
    first = 0.0 if case["fresh"] else 1.0
    s["conv_in"] = _randn(gen, (seqs, 3, ch)) * first
    s["delta_in"] = _randn(gen, (seqs, hv, 128, 128), std=0.05) * first
    return s


# ---- one pass ------------------------------------------------------------------------------------

def run(state):
    return (_own if own else _plain)[state["op"]](state)


def _library():
    if "nmoe_b200" not in sys.modules:
        sys.path.insert(0, os.path.join(os.getcwd(), "nano-metal-moe-qwen36_b200"))
    import nmoe_b200
    return nmoe_b200


def _own_attn(s):
    """The layer's handles and workspace, made at the first pass and kept by the program."""
    N, kept, c = _library(), s["kept"], s["case"]
    if not kept:
        kept["shape"] = N.FullAttnShape(c["q_heads"], c["kv_heads"], c["head_dim"], c["rotary"], True, THETA, EPS)
        kept["cache"] = N.PagedKV(s["k_pages"], s["v_pages"], s["table"])
        kept["weights"] = {"q_norm": s["q_norm"], "k_norm": s["k_norm"]}
        kept["dtype"] = N.DTYPE_BF16 if c["dtype"] == BF16 else N.DTYPE_F32
        need = 0
        if s["op"] == "step":
            need = N.full_attn_step_paged_workspace_bytes(kept["shape"], s["seqs"])
        elif s["op"] == "prefill":
            need = N.full_attn_prefill_paged_workspace_bytes(kept["shape"], s["seqs"], s["total"])
        kept["workspace"] = torch.empty(max(need, 16), dtype=torch.uint8, device="cuda")
    return N, kept, c


def _own_append(s):
    N, kept, _ = _own_attn(s)
    N.full_attn_append_paged(kept["weights"], kept["shape"], kept["cache"], s["k_new"], s["v_new"], s["cu_rows"],
                             s["kv_lens"], x_dtype=kept["dtype"])
    return {"k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def _own_step(s):
    N, kept, c = _own_attn(s)
    out = torch.empty(s["seqs"], c["q_heads"] * c["head_dim"], dtype=TORCH[c["dtype"]], device="cuda")
    N.full_attn_step_paged(kept["weights"], kept["shape"], kept["cache"], s["kv_lens"], s["q"], s["k_new"], s["v_new"],
                           out, kept["workspace"], x_dtype=kept["dtype"], out_dtype=kept["dtype"])
    return {"out": out, "k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def _own_prefill(s):
    N, kept, c = _own_attn(s)
    out = torch.empty(s["total"], c["q_heads"] * c["head_dim"], dtype=torch.bfloat16, device="cuda")
    N.full_attn_prefill_paged(kept["weights"], kept["shape"], kept["cache"], s["q"], s["cu_rows"], s["kv_lens"], out,
                              kept["workspace"], x_dtype=kept["dtype"])
    return {"out": out}


def _own_gdn(s):
    N, kept, c = _library(), s["kept"], s["case"]
    if not kept:
        kept["shape"] = N.LinearAttnShape(c["key_heads"], c["value_heads"])
        kept["weights"] = {k: s[k] for k in ("conv_w", "A_log", "dt_bias", "norm_w")}
        need = N.linear_attn_prefill_workspace_bytes(kept["shape"], s["seqs"], s["total"])
        kept["workspace"] = torch.empty(max(need, 16), dtype=torch.uint8, device="cuda")
    dtype = N.DTYPE_BF16 if c["dtype"] == BF16 else N.DTYPE_F32
    out = torch.empty(s["total"], c["value_heads"] * 128, dtype=TORCH[c["dtype"]], device="cuda")
    conv, delta = torch.empty_like(s["conv_in"]), torch.empty_like(s["delta_in"])
    N.linear_attn_prefill(kept["weights"], kept["shape"], s["qkv"], s["z"], s["alpha"], s["beta"], s["cu_rows"],
                          s["conv_in"], s["delta_in"], conv, delta, out, kept["workspace"], x_dtype=dtype,
                          out_dtype=dtype)
    return {"out": out, "conv": conv, "delta": delta}


_own = {"append": _own_append, "step": _own_step, "prefill": _own_prefill, "gdn": _own_gdn}


# ---- plain forms ---------------------------------------------------------------------------------

def _places(s):
    """Each packed row's sequence and position, on the device."""
    row = torch.arange(s["total"], dtype=torch.int32, device="cuda")
    seq = torch.searchsorted(s["cu_rows"][1:].contiguous(), row, right=True)
    return seq, (s["kv_lens"][seq] - s["cu_rows"][seq + 1] + row).long()


def _rotated(x, weight, position, rotary):
    """RMS norm by (weight + 1), then the rotate-half rotation of the first `rotary` dims; x [rows][heads][d]."""
    x = x.float()
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * (weight.float() + 1.0)
    h = rotary // 2
    if not h:
        return x
    freq = THETA ** (-2.0 * torch.arange(h, device=x.device, dtype=torch.float64) / rotary)
    angle = position.double()[:, None, None] * freq
    c, sn = angle.cos().float(), angle.sin().float()
    a, b = x[..., :h], x[..., h:rotary]
    return torch.cat([a * c - b * sn, a * sn + b * c, x[..., rotary:]], dim=-1)


def _plain_append(s):
    c = s["case"]
    hk, d, page = c["kv_heads"], c["head_dim"], c["page"]
    seq, position = _places(s)
    k = _rotated(s["k_new"].reshape(-1, hk, d), s["k_norm"], position, c["rotary"])
    where = s["table"][seq, position // page].long()
    s["k_pages"][where, position % page] = k.to(torch.bfloat16)
    s["v_pages"][where, position % page] = s["v_new"].reshape(-1, hk, d).to(torch.bfloat16)
    return {"k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def _plain_step(s):
    c = s["case"]
    hq, hk, d, page, n = c["q_heads"], c["kv_heads"], c["head_dim"], c["page"], s["seqs"]
    pages = _plain_append(s)
    q = s["q"].reshape(n, hq, 2, d)
    query = _rotated(q[:, :, 0], s["q_norm"], s["kv_lens"] - 1, c["rotary"]).reshape(n, hk, hq // hk, d)
    gather = lambda p: p[s["table"].long()].reshape(n, -1, hk, d).transpose(1, 2).float()  # noqa: E731
    score = query @ gather(s["k_pages"]).transpose(2, 3) / math.sqrt(d)
    hidden = torch.arange(score.shape[-1], device="cuda") >= s["kv_lens"][:, None]
    score.masked_fill_(hidden[:, None, None, :], -math.inf)
    p = torch.exp(score - score.amax(-1, keepdim=True))
    out = (p @ gather(s["v_pages"])) / p.sum(-1, keepdim=True)
    out = out.reshape(n, hq, d) * torch.sigmoid(q[:, :, 1].float())
    return {"out": out.reshape(n, hq * d).to(TORCH[c["dtype"]]), **pages}


def _plain_prefill(s):
    c = s["case"]
    hq, hk, d, page = c["q_heads"], c["kv_heads"], c["head_dim"], c["page"]
    _, position = _places(s)
    q = s["q"].reshape(-1, hq, 2, d)
    query = _rotated(q[:, :, 0], s["q_norm"], position, c["rotary"])
    out = torch.empty(s["total"], hq, d, device="cuda")
    at = 0
    for b, rows in enumerate(s["rows"]):   # packed sequences share nothing
        if rows == 0:
            continue
        length = s["lens"][b]
        table = s["table"][b, :-(-length // page)].long()
        k, v = (p[table].reshape(-1, hk, d)[:length].transpose(0, 1).float() for p in (s["k_pages"], s["v_pages"]))
        x = query[at:at + rows].reshape(rows, hk, -1, d).permute(1, 2, 0, 3).reshape(hk, -1, d)
        score = (x @ k.transpose(1, 2)).div_(math.sqrt(d)).view(hk, hq // hk, rows, length)
        score.masked_fill_(torch.arange(length, device="cuda") > position[at:at + rows, None], -math.inf)
        score.sub_(score.amax(-1, keepdim=True)).exp_()
        y = (score.view(hk, -1, length) @ v).view(hk, hq // hk, rows, d) / score.sum(-1, keepdim=True)
        out[at:at + rows] = y.permute(2, 0, 1, 3).reshape(rows, hq, d)
        at += rows
    out = out * torch.sigmoid(q[:, :, 1].float())
    return {"out": out.reshape(-1, hq * d).to(torch.bfloat16)}


CHUNK = 64


def _plain_gdn(s):
    """Chunks of 64 tokens: inside a chunk the rank-one updates are a triangular system, solved for all chunks at once."""
    c = s["case"]
    n, hk, hv, ch = s["seqs"], c["key_heads"], c["value_heads"], s["qkv"].shape[1]
    chunks = max(1, -(-max(s["rows"]) // CHUNK))
    row = torch.arange(s["total"], dtype=torch.int32, device="cuda")
    seq = torch.searchsorted(s["cu_rows"][1:].contiguous(), row, right=True)
    place = (row - s["cu_rows"][seq]).long()
    # the convolution over each sequence's own rows, its last three inputs in front
    x = torch.zeros(n, 3 + chunks * CHUNK, ch, device="cuda")
    x[:, :3] = s["conv_in"]
    x[seq, 3 + place] = s["qkv"].float()
    w = s["conv_w"].float()
    y = sum(x[:, j:j + chunks * CHUNK] * w[:, j] for j in range(4))
    y = y * torch.sigmoid(y)
    last = (s["cu_rows"][1:] - s["cu_rows"][:-1])[:, None] + torch.arange(3, device="cuda")
    conv = torch.gather(x, 1, last[:, :, None].expand(-1, -1, ch).long())
    live = torch.zeros(n, chunks * CHUNK, 1, device="cuda")
    live[seq, place] = 1.0

    def heads(t, h):   # [n][chunks * 64][h * 128] -> [n][hv][chunks][64][128]
        t = (t * live).view(n, chunks, CHUNK, h, 128).permute(0, 3, 1, 2, 4)
        return t.repeat_interleave(hv // h, 1)

    def scaled(t, by):
        t = t.reshape(n, -1, hk, 128)
        return (t * torch.rsqrt((t * t).mean(-1, keepdim=True) + 1e-12) * by).reshape(n, -1, hk * 128)

    q = heads(scaled(y[..., :hk * 128], 1 / 128), hk)
    k = heads(scaled(y[..., hk * 128:2 * hk * 128], 128 ** -0.5), hk)
    v = heads(y[..., 2 * hk * 128:], hv)
    dt = s["alpha"].float() + s["dt_bias"].float()
    rate = torch.zeros(n, chunks * CHUNK, hv, device="cuda")
    beta = torch.zeros_like(rate)
    rate[seq, place] = -torch.exp(s["A_log"]) * (torch.clamp(dt, min=0) + torch.log1p(torch.exp(-dt.abs())))
    beta[seq, place] = torch.sigmoid(s["beta"].float())
    rate, beta = (t.view(n, chunks, CHUNK, hv).permute(0, 3, 1, 2) for t in (rate, beta))
    g = rate.cumsum(-1)
    lower = torch.ones(CHUNK, CHUNK, device="cuda").tril().bool()
    decay = torch.exp((g[..., :, None] - g[..., None, :]).masked_fill(~lower, -math.inf))
    m = (beta[..., None] * decay * (k @ k.transpose(-1, -2))).masked_fill(torch.eye(CHUNK, device="cuda").bool(), 0.0)
    attend = decay * (q @ k.transpose(-1, -2))
    solve = torch.eye(CHUNK, device="cuda").expand_as(m).contiguous()
    for i in range(1, CHUNK):   # (I + m)^-1 by rows, every chunk at once
        solve[..., i:i + 1, :] -= m[..., i:i + 1, :i] @ solve[..., :i, :]
    state = s["delta_in"].clone()
    out = torch.empty_like(v)
    grow = torch.exp(g)[..., None]
    left = torch.exp(g[..., -1:] - g)[..., None]
    for j in range(chunks):   # the recurrence itself
        back = state.transpose(-1, -2)
        u = solve[:, :, j] @ (beta[:, :, j, :, None] * (v[:, :, j] - grow[:, :, j] * (k[:, :, j] @ back)))
        out[:, :, j] = grow[:, :, j] * (q[:, :, j] @ back) + attend[:, :, j] @ u
        state = state * grow[:, :, j, -1:] + (left[:, :, j] * u).transpose(-1, -2) @ k[:, :, j]
    o = out.permute(0, 2, 3, 1, 4).reshape(n, -1, hv, 128)[seq, place]
    o = o * torch.rsqrt((o * o).mean(-1, keepdim=True) + 1e-6) * s["norm_w"].float()
    z = s["z"].float()
    o = o.reshape(-1, hv * 128) * z * torch.sigmoid(z)
    return {"out": o.to(TORCH[c["dtype"]]), "conv": conv, "delta": state}


_plain = {"append": _plain_append, "step": _plain_step, "prefill": _plain_prefill, "gdn": _plain_gdn}


# ---- what a pass cannot do without ------------------------------------------------------------------

def work(case):
    rows = _lengths(case["rows"])
    total, size = sum(rows), 2 if case["dtype"] == BF16 else 4
    if case["op"] == "gdn":
        hk, hv = case["key_heads"], case["value_heads"]
        ch = (2 * hk + hv) * 128
        states = len(rows) * (3 * ch + hv * 128 * 128) * 4
        # a token and value head: S k, the update and S q, each 128 x 128
        return {"bytes": total * (ch + 2 * hv * 128 + 2 * hv) * size + 2 * states + ch * 8,
                "flops": total * hv * 128 * 128 * 6}
    hq, hk, d = case["q_heads"], case["kv_heads"], case["head_dim"]
    past = _lengths(case["past"])
    new = total * hk * d * 2 * (size + 2)   # the new keys and values, read and written
    if case["op"] == "append":
        return {"bytes": new, "flops": total * hk * d * 8}
    if case["op"] == "step":
        seen = sum(p + 1 for p in past)
        return {"bytes": new + sum(past) * hk * d * 4 + total * hq * d * 3 * size, "flops": seen * hq * d * 4}
    seen = sum(n * p + n * (n + 1) // 2 for n, p in zip(rows, past))
    read = sum(n + p for n, p in zip(rows, past) if n)
    return {"bytes": read * hk * d * 4 + total * hq * d * (2 * size + 2), "flops": seen * hq * d * 4}


# ---- from the definitions, in 64 bits ----------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "step": _exact_step, "prefill": _exact_prefill, "gdn": _exact_gdn}[s["op"]](s)


def _turn64(x, weight, at, rotary):
    """One row's heads [heads][d] in 64 bits at position `at`: unit mean square, the weights, then each
    pair (t, t + rotary / 2) turned as a complex number."""
    x = x.double()
    x = x / torch.sqrt(torch.mean(x ** 2, -1, keepdim=True) + EPS) * (1 + weight.double())
    h = rotary // 2
    if h:
        turn = torch.arange(h, dtype=torch.float64, device=x.device) * (-2 * math.log(THETA) / rotary)
        pair = torch.complex(x[..., :h], x[..., h:rotary]) * torch.polar(torch.ones_like(turn), at.double()[..., None, None] * turn.exp())
        x = torch.cat([pair.real, pair.imag, x[..., rotary:]], -1)
    return x


def _exact_rows(s, b):
    """Sequence b's first row, its positions, and its pages' rows in order."""
    c = s["case"]
    first, rows, length = sum(s["rows"][:b]), s["rows"][b], s["lens"][b]
    at = torch.arange(length - rows, length, device="cuda")
    places = s["table"][b].long().repeat_interleave(c["page"])[:length], torch.arange(length, device="cuda") % c["page"]
    return first, rows, at, places


def _exact_append(s):
    c = s["case"]
    hk, d = c["kv_heads"], c["head_dim"]
    for b in range(s["seqs"]):
        first, rows, at, (page, slot) = _exact_rows(s, b)
        if rows:
            k = _turn64(s["k_new"][first:first + rows].reshape(rows, hk, d), s["k_norm"], at, c["rotary"])
            s["k_pages"][page[-rows:], slot[-rows:]] = k.to(torch.bfloat16)
            s["v_pages"][page[-rows:], slot[-rows:]] = s["v_new"][first:first + rows].reshape(rows, hk, d).to(torch.bfloat16)
    return {"k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def _exact_attention(s):
    c = s["case"]
    hq, hk, d = c["q_heads"], c["kv_heads"], c["head_dim"]
    out = torch.zeros(s["total"], hq, d, dtype=torch.float64, device="cuda")
    for b in range(s["seqs"]):
        first, rows, at, places = _exact_rows(s, b)
        if not rows:
            continue
        q = s["q"][first:first + rows].reshape(rows, hq, 2 * d)
        query, gate = _turn64(q[..., :d], s["q_norm"], at, c["rotary"]), 1 / (1 + torch.exp(-q[..., d:].double()))
        k, v = s["k_pages"][places].double(), s["v_pages"][places].double()
        for h in range(hq):
            for r in range(0, rows, 4096):
                dots = query[r:r + 4096, h] @ k[:, h * hk // hq].T * d ** -0.5
                dots[torch.arange(len(k), device="cuda")[None] > at[r:r + 4096, None]] = -math.inf
                out[first + r:first + min(r + 4096, rows), h] = torch.softmax(dots, -1) @ v[:, h * hk // hq]
        out[first:first + rows] *= gate
    return out.reshape(-1, hq * d)


def _exact_step(s):
    pages = _exact_append(s)
    return {"out": _exact_attention(s), **pages}


def _exact_prefill(s):
    return {"out": _exact_attention(s)}


def _exact_gdn(s):
    """The recurrence token by token, all heads of a sequence together."""
    c = s["case"]
    hk, hv = c["key_heads"], c["value_heads"]
    w, rate = s["conv_w"].double(), -torch.exp(s["A_log"].double())
    out = torch.zeros(s["total"], hv, 128, dtype=torch.float64, device="cuda")
    conv, delta = s["conv_in"].double().clone(), s["delta_in"].double().clone()
    for b in range(s["seqs"]):
        first, rows = sum(s["rows"][:b]), s["rows"][b]
        if not rows:
            continue
        x = torch.cat([conv[b], s["qkv"][first:first + rows].double()])
        y = torch.nn.functional.conv1d(x.T[None], w[:, None, :], groups=len(w))[0].T
        y = y / (1 + torch.exp(-y))
        q, k, v = (t.reshape(rows, -1, 128) for t in y.split([hk * 128, hk * 128, hv * 128], 1))
        q = q / torch.sqrt(torch.mean(q ** 2, -1, keepdim=True) + 1e-12) / 128
        k = k / torch.sqrt(torch.mean(k ** 2, -1, keepdim=True) + 1e-12) / math.sqrt(128)
        q, k = q.repeat_interleave(hv // hk, 1), k.repeat_interleave(hv // hk, 1)
        keep = torch.exp(rate * torch.logaddexp(s["alpha"][first:first + rows].double() + s["dt_bias"].double(), torch.zeros((), dtype=torch.float64, device="cuda")))
        beta = 1 / (1 + torch.exp(-s["beta"][first:first + rows].double()))
        state = delta[b]
        for t in range(rows):
            state = state * keep[t, :, None, None]
            miss = (v[t] - (state @ k[t, :, :, None])[..., 0]) * beta[t, :, None]
            state = state + miss[:, :, None] * k[t, :, None, :]
            out[first + t] = (state @ q[t, :, :, None])[..., 0]
        o, z = out[first:first + rows], s["z"][first:first + rows].double().reshape(rows, hv, 128)
        o /= torch.sqrt(torch.mean(o ** 2, -1, keepdim=True) + 1e-6)
        o *= s["norm_w"].double() * z / (1 + torch.exp(-z))
        conv[b], delta[b] = x[-3:], state
    return {"out": out.reshape(-1, hv * 128), "conv": conv, "delta": delta}
