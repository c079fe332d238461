"""64-bit statements of the prompt and paged-cache attention operators, and inputs for their
tests. torch float64 on the tensors' own device, sequence by sequence, head by head."""
import math

import torch

THETA, EPS = 1e7, 1e-6


def rotate(x, position, rotary, theta=THETA):
    """x [rows][heads][d] float64, position [rows]: dims t and t + rotary / 2 turned together."""
    h = rotary // 2
    if h == 0:
        return x
    t = torch.arange(h, dtype=torch.float64, device=x.device)
    ang = position.double()[:, None, None] * theta ** (-2.0 * t / rotary)
    a, b = x[..., :h], x[..., h:rotary]
    return torch.cat([a * ang.cos() - b * ang.sin(), a * ang.sin() + b * ang.cos(), x[..., rotary:]], -1)


def prepared(x, weight, position, rotary):
    x = x.double()
    if weight is not None:
        x = x / (x.pow(2).mean(-1, keepdim=True) + EPS).sqrt() * (weight.double() + 1)
    return rotate(x, position, rotary)


class Packed:
    """A packed batch over a paged cache: rows and past lengths per sequence."""

    def __init__(self, rows, past, page, q_heads, kv_heads, d, rotary, dtype=torch.bfloat16, order="rows", fused=False,
                 gated=True, norm=True, seed=0, spare_rows=0, tail=None, device="cuda"):
        g = torch.Generator(device=device).manual_seed(seed)
        rnd = lambda *s, std=1.0: torch.randn(s, generator=g, device=device) * std  # noqa: E731
        self.rows, self.past, self.page, self.hq, self.hk, self.d, self.rotary = rows, past, page, q_heads, kv_heads, d, rotary
        self.gated, self.dtype = gated, dtype
        self.lens = [a + b for a, b in zip(rows, past)]
        self.total = sum(rows) + spare_rows
        self.cu = torch.tensor([sum(rows[:i]) for i in range(len(rows) + 1)], dtype=torch.int32, device=device)
        self.kv_lens = torch.tensor(self.lens, dtype=torch.int32, device=device)
        need = [max(0, -(-n // page)) for n in self.lens]
        pages = sum(need) + 4
        perm = torch.randperm(pages, generator=g, device=device).to(torch.int32)
        self.table = torch.full((len(rows), max(1, max(need)) + 1), -1, dtype=torch.int32, device=device)
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = perm[at:at + n]
            at += n
        shape = (pages, page, kv_heads, d) if order == "rows" else (pages, kv_heads, page, d)
        k, v = (rnd(*shape).to(torch.bfloat16) for _ in range(2))
        if order != "rows":
            k, v = k.transpose(1, 2), v.transpose(1, 2)
        self.k, self.v = k, v
        if tail is not None:   # what no position uses
            used = torch.zeros(pages, page, dtype=torch.bool, device=device)
            for b, n in enumerate(self.lens):
                p = torch.arange(max(0, n), device=device)
                used[self.table[b, p // page].long(), p % page] = True
            for t in (k, v):
                t[~used] = tail
        wide = [q_heads * d * (2 if gated else 1), kv_heads * d, kv_heads * d]
        if fused:
            self.q, self.k_new, self.v_new = rnd(self.total, sum(wide)).to(dtype).split(wide, 1)
        else:
            self.q, self.k_new, self.v_new = (rnd(self.total, w).to(dtype) for w in wide)
        self.weights = {n: rnd(d, std=0.1).to(torch.bfloat16) if norm else None for n in ("q_norm", "k_norm")}

    def places(self, b):
        """Device indices (page, row) of positions 0 .. len - 1 of sequence b; -1: no page."""
        p = torch.arange(self.lens[b], device=self.table.device)
        return self.table[b, p // self.page].long(), p % self.page

    def append(self):
        """(k, v) the pages should hold, in float64: unrounded new keys, rounded values."""
        k, v = self.k.double().clone(), self.v.double().clone()
        for b, n in enumerate(self.rows):
            r0, first = int(self.cu[b]), self.lens[b] - n
            for_rows = torch.arange(max(0, -first), n, device=k.device)
            if len(for_rows) == 0:
                continue
            pos = first + for_rows
            new = prepared(self.k_new[r0 + for_rows].reshape(-1, self.hk, self.d), self.weights["k_norm"], pos, self.rotary)
            page, slot = self.places(b)
            k[page[pos], slot[pos]] = new
            v[page[pos], slot[pos]] = self.v_new[r0 + for_rows].reshape(-1, self.hk, self.d).to(torch.bfloat16).double()
        return k, v

    def attention(self, scale=None):
        """(out, mass, reach): the attention of every row over the pages as they are, float64; mass: sum of
        p |v| times the gate; reach: the largest sum of |q k| scale of a row and head."""
        out = torch.zeros(self.total, self.hq, self.d, dtype=torch.float64, device=self.q.device)
        mass, reach = torch.zeros_like(out), torch.zeros(self.total, self.hq, 1, dtype=torch.float64, device=self.q.device)
        scale = scale or self.d ** -0.5
        for b, n in enumerate(self.rows):
            r0 = int(self.cu[b])
            if n == 0 or self.lens[b] <= 0:
                continue
            pos = torch.arange(self.lens[b] - n, self.lens[b], device=self.q.device)
            q = self.q[r0:r0 + n].reshape(n, self.hq, -1)
            x = prepared(q[..., :self.d], self.weights["q_norm"], pos, self.rotary)
            gate = torch.sigmoid(q[..., self.d:].double()) if self.gated else torch.ones_like(x)
            page, slot = self.places(b)
            no_page = (page < 0) | (page >= self.k.shape[0])
            page = page.clamp(0, self.k.shape[0] - 1)
            k, v = self.k[page, slot].double(), self.v[page, slot].double()
            hidden = (torch.arange(self.lens[b], device=pos.device)[None] > pos[:, None]) | no_page[None]
            k, v = k.masked_fill(no_page[:, None, None], 0), v.masked_fill(no_page[:, None, None], 0)
            for h in range(self.hq):
                kh = h // (self.hq // self.hk)
                s = (x[:, h] @ k[:, kh].T * scale).masked_fill(hidden, -math.inf)
                p = torch.exp(s - s.amax(-1, keepdim=True).clamp(min=-1e300))
                p = p / p.sum(-1, keepdim=True).clamp(min=1e-300)
                out[r0:r0 + n, h] = p @ v[:, kh] * gate[:, h]
                mass[r0:r0 + n, h] = p @ v[:, kh].abs() * gate[:, h]
                reach[r0:r0 + n, h, 0] = (x[:, h].abs() @ k[:, kh].abs().T * scale).masked_fill(hidden, 0).amax(-1)
        return out, mass, reach


def gdn(w, hk, hv, cu, qkv, z, alpha, beta, conv, delta):
    """The GatedDeltaNet core token by token in float64; conv / delta (float64) updated in place."""
    cw, nw = w["conv_w"].double(), w["norm_w"].double()
    out = torch.zeros(qkv.shape[0], hv * 128, dtype=torch.float64, device=qkv.device)
    for b in range(len(cu) - 1):
        for r in range(cu[b], cu[b + 1]):
            x = torch.cat([conv[b], qkv[r].double()[None]])
            y = (x * cw.T).sum(0)
            y = y * torch.sigmoid(y)
            conv[b] = x[1:]
            q, k, v = y[:hk * 128].view(hk, 128), y[hk * 128:2 * hk * 128].view(hk, 128), y[2 * hk * 128:].view(hv, 128)
            q = q / (q.pow(2).mean(-1, keepdim=True) + 1e-12).sqrt() / 128
            k = k / (k.pow(2).mean(-1, keepdim=True) + 1e-12).sqrt() / math.sqrt(128)
            q, k = q.repeat_interleave(hv // hk, 0), k.repeat_interleave(hv // hk, 0)
            dt = alpha[r].double() + w["dt_bias"].double()
            g = torch.exp(-torch.exp(w["A_log"].double()) * torch.logaddexp(dt, torch.zeros_like(dt)))
            s = delta[b] * g[:, None, None]
            d = (v - (s @ k[:, :, None])[..., 0]) * torch.sigmoid(beta[r].double())[:, None]
            s = s + d[:, :, None] * k[:, None, :]
            delta[b] = s
            o = (s @ q[:, :, None])[..., 0]
            o = o / (o.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt() * nw
            zz = z[r].double().view(hv, 128)
            out[r] = (o * zz * torch.sigmoid(zz)).reshape(-1)
    return out
