"""What the binding of the prompt and paged-cache calls refuses, on CPU tensors: the device check is
told that the host is the current device, and no call of the library is reached."""
import pytest
import torch

import nmoe_b200 as N


class Unreached:
    """The library without its kernels: what computes a size works, any other call is a failure."""

    def __init__(self, real):
        self.real = real

    def __getattr__(self, name):
        if name.endswith("_workspace_bytes"):
            return getattr(self.real, name)
        raise AssertionError(f"{name} was called")


@pytest.fixture
def on_host(monkeypatch):
    real = N.lib()
    monkeypatch.setitem(N._dtypes(), "device", lambda: -1)
    monkeypatch.setattr(N, "lib", lambda: Unreached(real))


def bf16(*shape):
    return torch.zeros(shape, dtype=torch.bfloat16)


def i32(*values):
    return torch.tensor(values, dtype=torch.int32)


SHAPE = N.FullAttnShape(4, 2, 128, 64, False)
LINEAR = N.LinearAttnShape(1, 2)
ROWS = 6


def operands():
    """Each call's operands by name, packed rows of ROWS rows."""
    return {
        "append": {"k_new": bf16(ROWS, 256), "v_new": bf16(ROWS, 256)},
        "prefill": {"q": bf16(ROWS, 512), "workspace": torch.zeros(1 << 20, dtype=torch.uint8)},
        "step": {"q": bf16(ROWS, 512), "k_new": bf16(ROWS, 256), "v_new": bf16(ROWS, 256),
                 "workspace": torch.zeros(1 << 22, dtype=torch.uint8)},
        "linear": {"qkv": bf16(ROWS, 512), "z": bf16(ROWS, 256), "alpha": bf16(ROWS, 2), "beta": bf16(ROWS, 2),
                   "workspace": torch.zeros(1 << 20, dtype=torch.uint8)},
    }


def cache(seqs):
    return N.PagedKV(bf16(4, 16, 2, 128), bf16(4, 16, 2, 128), torch.zeros(seqs, 2, dtype=torch.int32))


def call(name, x):
    if name == "append":
        N.full_attn_append_paged({}, SHAPE, cache(1), x["k_new"], x["v_new"], i32(0, ROWS), i32(ROWS))
    elif name == "prefill":
        N.full_attn_prefill_paged({}, SHAPE, cache(1), x["q"], i32(0, ROWS), i32(ROWS), bf16(ROWS, 512), x["workspace"])
    elif name == "step":
        N.full_attn_step_paged({}, SHAPE, cache(ROWS), i32(*[1] * ROWS), x["q"], x["k_new"], x["v_new"], bf16(ROWS, 512),
                               x["workspace"], x_dtype=N.DTYPE_BF16, out_dtype=N.DTYPE_BF16)
    else:
        w = {"conv_w": bf16(512, 4), "A_log": torch.zeros(2), "dt_bias": bf16(2), "norm_w": bf16(128)}
        N.linear_attn_prefill(w, LINEAR, x["qkv"], x["z"], x["alpha"], x["beta"], i32(0, ROWS), None, None,
                              torch.zeros(1, 3, 512), torch.zeros(1, 2, 128, 128), bf16(ROWS, 256), x["workspace"])


@pytest.mark.parametrize("name", ["append", "prefill", "step", "linear"])
def test_plain_operands_reach_the_library(on_host, name):
    with pytest.raises(AssertionError, match="was called"):
        call(name, operands()[name])


BROADCAST = [("append", ["k_new"]), ("append", ["v_new"]), ("append", ["k_new", "v_new"]), ("prefill", ["q"]),
             ("step", ["q"]), ("step", ["k_new", "v_new"]), ("linear", ["qkv"]), ("linear", ["z"]),
             ("linear", ["alpha", "beta"])]


@pytest.mark.parametrize("name,which", BROADCAST, ids=lambda x: x if isinstance(x, str) else "+".join(x))
@pytest.mark.parametrize("heads", [False, True], ids=["2d", "3d"])
def test_broadcast_rows_are_refused(on_host, name, which, heads):
    """A row expanded over all rows has stride 0, which the library takes for packed rows."""
    x = operands()[name]
    for n in which:
        t = x[n][:1].view(1, 2, -1).expand(ROWS, -1, -1) if heads else x[n][:1].expand(ROWS, -1)
        x[n] = t
    with pytest.raises(N.NmoeError) as e:
        call(name, x)
    assert e.value.status == N.EINVAL


@pytest.mark.parametrize("stride", [1, 8, 255])
def test_overlapping_rows_are_refused(on_host, stride):
    x = bf16(ROWS, 256).view(-1).as_strided((ROWS, 256), (stride, 1))
    with pytest.raises(N.NmoeError) as e:
        call("append", {"k_new": x, "v_new": x})
    assert e.value.status == N.EINVAL


def test_one_row_has_any_stride(on_host):
    """One row is read whatever its stride says: a row of a wider tensor, an expanded one."""
    wide = bf16(3, 1024)
    for t in (wide[1:2, :256], wide[:1, :256].expand(1, -1), wide[:, 256:512][2:3]):
        assert N._rows(t, 1, 256, N.DTYPE_BF16, "x") == 256
    assert N._rows(wide[:, :256], 3, 256, N.DTYPE_BF16, "x") == 1024
    assert N._rows(wide[:, :256].unflatten(1, (2, 128)), 3, 256, N.DTYPE_BF16, "x") == 1024


@pytest.mark.parametrize("name", ["prefill", "step", "linear"])
def test_workspaces_with_holes_are_refused(on_host, name):
    """A workspace counts as large as its elements only when they lie together."""
    x = operands()[name]
    n = x["workspace"].numel()
    for t in (torch.zeros(1, dtype=torch.uint8).expand(n), torch.zeros(8, dtype=torch.uint8)[::2].expand(n // 4, 4)):
        x["workspace"] = t
        with pytest.raises(N.NmoeError) as e:
            call(name, x)
        assert e.value.status == N.EINVAL


class Elsewhere(torch.Tensor):
    """A tensor that says it is on device 5."""

    def get_device(self):
        return 5


@pytest.mark.parametrize("name", ["append", "prefill", "step"])
def test_a_cache_of_another_device_is_refused(on_host, monkeypatch, name):
    """The cache is checked at the call, not only where it was made: the current device may be another one by then."""
    monkeypatch.setitem(N._dtypes(), "device", lambda: 5)
    seqs = ROWS if name == "step" else 1
    far = N.PagedKV(*(bf16(4, 16, 2, 128).as_subclass(Elsewhere) for _ in range(2)),
                    torch.zeros(seqs, 2, dtype=torch.int32).as_subclass(Elsewhere))
    monkeypatch.setitem(N._dtypes(), "device", lambda: -1)
    monkeypatch.setitem(globals(), "cache", lambda n: far)
    with pytest.raises(N.NmoeError) as e:
        call(name, operands()[name])
    assert e.value.status == N.EINVAL
