"""What the prompt and paged-cache calls refuse, on the host: no argument here reaches a GPU."""
import ctypes as C

import pytest

import nmoe_b200 as N

A = 0x10000   # an aligned address that is never read


def attn(**kw):
    """A valid argument set with changes, for the three paged calls."""
    a = dict(q_heads=16, kv_heads=2, head_dim=256, rotary=64, gated=1, theta=1e7, eps=1e-6, norm=A, pages=10,
             page_size=16, max_pages=4, ps=8192, rs=512, hs=256, k=A, v=A, table=A, ts=4, x_dtype=N.DTYPE_BF16,
             out_dtype=N.DTYPE_BF16, q=A, k_new=A, v_new=A, cu=A, lens=A, out=A, ws=A, qs=0, kvs=0, scale=0.0, n=2, rows=5)
    a.update(kw)
    w = N.FullAttnWeights(a["norm"], a["norm"])
    s = N.FullAttnShape(a["q_heads"], a["kv_heads"], a["head_dim"], a["rotary"], True, a["theta"], a["eps"])
    s.gated = a["gated"]
    c = N.PagedKVHost(a["k"], a["v"], a["ps"], a["rs"], a["hs"], a["pages"], a["page_size"], a["table"], a["max_pages"],
                      a["ts"])
    return a, C.byref(w), C.byref(s), C.byref(c)


def calls(**kw):
    L = N.lib()
    a, w, s, c = attn(**kw)
    yield "append", lambda: L.nmoe_full_attn_append_paged(w, s, c, a["n"], a["rows"], a["cu"], a["lens"], a["k_new"],
                                                          a["v_new"], a["x_dtype"], a["kvs"], None)
    yield "prefill", lambda: L.nmoe_full_attn_prefill_paged(w, s, c, a["n"], a["rows"], a["cu"], a["lens"], a["q"],
                                                            a["x_dtype"], a["qs"], a["scale"], a["out"], a["ws"], None)
    yield "step", lambda: L.nmoe_full_attn_step_paged(w, s, c, a["n"], a["lens"], a["q"], a["qs"], a["k_new"], a["v_new"],
                                                      a["kvs"], a["x_dtype"], a["scale"], a["out"], a["out_dtype"],
                                                      a["ws"], None)


ALL = ["append", "prefill", "step"]
REFUSED = [
    (dict(head_dim=64), ALL), (dict(head_dim=192), ALL), (dict(q_heads=15), ALL), (dict(q_heads=18), ALL),
    (dict(kv_heads=0), ALL), (dict(rotary=48), ALL), (dict(rotary=8), ALL), (dict(rotary=512), ALL), (dict(rotary=-16), ALL),
    (dict(theta=0.0), ALL), (dict(theta=float("nan")), ALL), (dict(eps=0.0), ALL), (dict(eps=float("nan")), ALL),
    (dict(gated=2), ALL), (dict(pages=0), ALL), (dict(page_size=0), ALL), (dict(max_pages=0), ALL),
    (dict(max_pages=1 << 27), ALL), (dict(page_size=1, max_pages=(1 << 31) - 256), ALL), (dict(k=None), ALL), (dict(v=None), ALL), (dict(table=None), ALL), (dict(table=A + 2), ALL),
    (dict(k=A + 8), ALL), (dict(ps=8193), ALL), (dict(rs=4), ALL), (dict(hs=-256), ALL), (dict(ts=-1), ALL),
    (dict(x_dtype=N.DTYPE_Q4), ALL), (dict(n=-1), ALL), (dict(lens=None), ALL),
    (dict(rows=-1), ["append", "prefill"]), (dict(cu=None), ["append", "prefill"]), (dict(cu=A + 1), ["append", "prefill"]),
    (dict(k_new=None), ["append", "step"]), (dict(v_new=None), ["append", "step"]), (dict(k_new=A + 4), ["append", "step"]),
    (dict(kvs=500), ["append", "step"]), (dict(kvs=516), ["append", "step"]),
    (dict(q=None), ["prefill", "step"]), (dict(q=A + 8), ["prefill", "step"]), (dict(qs=8190), ["prefill", "step"]),
    (dict(qs=8196), ["prefill", "step"]), (dict(out=None), ["prefill", "step"]), (dict(out=A + 2), ["prefill", "step"]),
    (dict(scale=-1.0), ["prefill", "step"]), (dict(scale=float("nan")), ["prefill", "step"]),
    (dict(scale=float("inf")), ["prefill", "step"]), (dict(ws=None), ["step"]), (dict(ws=A + 8), ["step"]),
    (dict(out_dtype=N.DTYPE_Q2), ["step"]),
]


@pytest.mark.parametrize("change,by", REFUSED, ids=[",".join(f"{k}={v}" for k, v in c.items()) for c, _ in REFUSED])
def test_attention_refusals(change, by):
    for name, call in calls(**change):
        if name in by:
            assert call() == N.EINVAL, name
            assert N.lib().nmoe_full_attn_error(), name


def test_null_structs():
    L = N.lib()
    for miss in range(3):
        a, *ptr = attn()
        ptr[miss] = None
        assert L.nmoe_full_attn_append_paged(*ptr, 1, 1, A, A, A, A, N.DTYPE_BF16, 0, None) == N.EINVAL
        assert L.nmoe_full_attn_prefill_paged(*ptr, 1, 1, A, A, A, N.DTYPE_BF16, 0, 0.0, A, A, None) == N.EINVAL
        assert L.nmoe_full_attn_step_paged(*ptr, 1, A, A, 0, A, A, 0, N.DTYPE_BF16, 0.0, A, N.DTYPE_BF16, A, None) == N.EINVAL


def test_nothing_to_do_is_no_error():
    for name, call in calls(n=0):
        assert call() == N.OK, name
    for name, call in calls(rows=0):
        if name != "step":
            assert call() == N.OK, name


def test_workspace_sizes():
    s = N.FullAttnShape(16, 2, 256, 64)
    assert N.full_attn_step_paged_workspace_bytes(s, 64) > N.full_attn_step_paged_workspace_bytes(s, 1) > 0
    assert N.full_attn_step_paged_workspace_bytes(s, 0) == 0
    assert N.full_attn_step_paged_workspace_bytes(N.FullAttnShape(16, 3), 4) == 0
    assert N.full_attn_prefill_paged_workspace_bytes(N.FullAttnShape(16, 3), 4, 100) == 0


def linear(**kw):
    a = dict(hk=16, hv=32, n=2, rows=5, cu=A, qkv=A, qs=0, z=A, zs=0, alpha=A, beta=A, abs=0, x_dtype=N.DTYPE_BF16,
             conv_in=A, delta_in=A, conv_out=A, delta_out=A, out=A, out_dtype=N.DTYPE_BF16, ws=A, conv_w=A, A_log=A,
             dt_bias=A, norm_w=A)
    a.update(kw)
    w = N.LinearAttnWeights(a["conv_w"], a["A_log"], a["dt_bias"], a["norm_w"])
    s = N.LinearAttnShape(a["hk"], a["hv"])
    return N.lib().nmoe_linear_attn_prefill(C.byref(w), C.byref(s), a["n"], a["rows"], a["cu"], a["qkv"], a["qs"], a["z"],
                                            a["zs"], a["alpha"], a["beta"], a["abs"], a["x_dtype"], a["conv_in"],
                                            a["delta_in"], a["conv_out"], a["delta_out"], a["out"], a["out_dtype"],
                                            a["ws"], None)


@pytest.mark.parametrize("change", [
    dict(hk=0), dict(hk=3), dict(hv=0), dict(hk=-16, hv=-32), dict(n=-1), dict(n=70000), dict(rows=-1), dict(cu=None),
    dict(cu=A + 2), dict(qkv=None), dict(z=None), dict(alpha=None), dict(beta=None), dict(out=None), dict(conv_out=None),
    dict(delta_out=None), dict(conv_w=None), dict(A_log=None), dict(dt_bias=None), dict(norm_w=None), dict(conv_w=A + 4),
    dict(x_dtype=N.DTYPE_Q4), dict(out_dtype=N.DTYPE_Q2), dict(qs=8000), dict(qs=8196), dict(zs=4095), dict(abs=31),
    dict(qkv=A + 8), dict(z=A + 4), dict(delta_in=A + 4), dict(delta_out=A + 8), dict(conv_in=A + 4), dict(out=A + 8)],
    ids=lambda c: ",".join(f"{k}={v}" for k, v in c.items()))
def test_linear_refusals(change):
    assert linear(**change) == N.EINVAL
    assert N.lib().nmoe_linear_attn_error()


def test_linear_nothing_to_do():
    assert linear(n=0) == N.OK


def test_tensors_off_the_gpu_are_refused():
    import torch
    k = torch.zeros(4, 16, 2, 256, dtype=torch.bfloat16)
    with pytest.raises(N.NmoeError):
        N.PagedKV(k, k, torch.zeros(1, 4, dtype=torch.int32))
    with pytest.raises(N.NmoeError):
        N.linear_attn_prefill({}, N.LinearAttnShape(1, 1), torch.zeros(4, 384), torch.zeros(4, 128), torch.zeros(4, 1),
                              torch.zeros(4, 1), torch.tensor([0, 4], dtype=torch.int32), None, None,
                              torch.zeros(1, 3, 384), torch.zeros(1, 1, 128, 128), torch.zeros(4, 128), None)
