"""The attention operators without a GPU: argument checks of the C ABI and of the Python entry points, and the rotation table."""
import math

import pytest
import torch

import ternary_vllm_amd as tv
from ternary_vllm_amd import attention_ops as A

lib = tv.custom_ops_mod._lib
P = 1 << 20      # an aligned address that is never read: every call below fails before a launch, or has nothing to launch


def attention_args(**kw):
    f = dict(size=A._ATTENTION.size, q=P, k=P, v=P, out=P, lse=P, slopes=0, prefix=0, documents=0, cache_len=0, count=0,
             batch=2, queries=3, keys=5, heads=4, kv_heads=2, dim=64)
    f.update({n: 0 for n in ("q_batch", "q_token", "q_head", "k_batch", "k_token", "k_head", "v_batch", "v_token", "v_head")})
    f.update(o_batch=3 * 4 * 64, o_token=4 * 64, o_head=64, prefix_value=0, documents_batch=0, cache_len_stride=0, cache_len_value=0,
             scale=0.125, softcap=0.0, dtype=1, causal=0)
    assert not set(kw) - set(f)
    f.update(kw)
    return A._ATTENTION.pack(*f.values())


def grads_args(**kw):
    f = dict(size=A._GRADS.size, grad_out=P, dq=P, dk=P, dv=P, g_batch=0, g_token=0, g_head=0)
    f.update(kw)
    return A._GRADS.pack(*f.values())


BAD = [(dict(size=8), "size"), (dict(dtype=3), "dtype"), (dict(batch=-1), "negative"), (dict(keys=-1), "negative"), (dict(heads=3), "multiple"), (dict(kv_heads=0), "multiple"),
       (dict(dim=0), "head dim"), (dict(dim=129), "head dim"), (dict(queries=1 << 31), "too"), (dict(batch=1 << 20, heads=1 << 14, kv_heads=1), "too many"),
       (dict(scale=math.nan), "scale"), (dict(scale=math.inf), "scale"), (dict(softcap=-1.0), "softcap"), (dict(softcap=math.nan), "softcap"), (dict(softcap=math.inf), "softcap"),
       (dict(q=0), "NULL"), (dict(out=0), "NULL"), (dict(k=0), "NULL"), (dict(v=0), "NULL"), (dict(q=P + 1), "misaligned"), (dict(lse=P + 2), "misaligned"),
       (dict(slopes=P + 2), "misaligned"), (dict(prefix=P + 4), "misaligned"), (dict(count=P + 4), "misaligned"), (dict(o_batch=0), "overlap"), (dict(o_head=32), "overlap")]


@pytest.mark.parametrize("kw,word", BAD)
def test_attention_refusals(kw, word):
    a = attention_args(**kw)
    for call in (lambda: lib.tvl_attention(a, None, 0, None), lambda: lib.tvl_cached_attention(a, None, 0, None), lambda: lib.tvl_attention_backward(a, grads_args(), P, 1 << 40, None)):
        assert call() == 1 and word in lib.tvl_last_error().decode(), lib.tvl_last_error()


def test_attention_refuses_missing_blocks_and_workspace():
    assert lib.tvl_attention(None, None, 0, None) == 1 and lib.tvl_cached_attention(None, None, 0, None) == 1
    a = attention_args()
    assert lib.tvl_attention(attention_args(documents=P), None, 0, None) == 1 and b"documents" in lib.tvl_last_error()
    assert lib.tvl_attention_backward(a, None, P, 1 << 40, None) == 1
    assert lib.tvl_attention_backward(a, grads_args(size=1), P, 1 << 40, None) == 1
    assert lib.tvl_attention_backward(a, grads_args(grad_out=0), P, 1 << 40, None) == 1 and b"NULL" in lib.tvl_last_error()
    assert lib.tvl_attention_backward(a, grads_args(dk=0), P, 1 << 40, None) == 1 and b"together" in lib.tvl_last_error()
    assert lib.tvl_attention_backward(attention_args(lse=0), grads_args(), P, 1 << 40, None) == 1
    need = lib.tvl_attention_backward_workspace_bytes(a)
    assert need > 0
    for ws, n in ((None, need), (P, need - 1), (P + 16, need)):
        assert lib.tvl_attention_backward(a, grads_args(), ws, n, None) == 1 and b"workspace" in lib.tvl_last_error()
    # nothing to do: no launch
    for fn in (lib.tvl_attention, lib.tvl_cached_attention):
        assert fn(attention_args(batch=0, q=0, k=0, v=0, out=0), None, 0, None) == 0
        assert fn(attention_args(queries=0, q=0, out=0), None, 0, None) == 0
    assert lib.tvl_attention_backward(attention_args(batch=0), grads_args(), None, 0, None) == 0


@pytest.mark.parametrize("kw", [dict(heads=1), dict(heads=3), dict(heads=0), dict(kv_heads=0), dict(kv_heads=-1), dict(batch=-1), dict(queries=-1), dict(keys=-1), dict(dim=0), dict(dim=-1),
                                dict(size=8)])
def test_workspaces_of_sizes_that_make_no_sense(kw):
    """A caller asks for a workspace before any check: no division by zero, no size, and the call itself is refused."""
    a = attention_args(documents=P, **kw)
    for name in ("attention", "attention_backward", "cached_attention"):
        assert getattr(lib, f"tvl_{name}_workspace_bytes")(a) == 0
        assert getattr(lib, f"tvl_{name}_workspace_bytes")(None) == 0
    assert lib.tvl_attention(a, None, 0, None) == 1 and lib.tvl_cached_attention(a, None, 0, None) == 1


@pytest.mark.parametrize("name", ["q_token", "k_token", "v_token"])
def test_negative_token_strides_are_refused(name):
    a = attention_args(**{name: -64})
    for call in (lambda: lib.tvl_attention(a, None, 0, None), lambda: lib.tvl_cached_attention(a, None, 0, None), lambda: lib.tvl_attention_backward(a, grads_args(), P, 1 << 40, None)):
        assert call() == 1 and b"stride" in lib.tvl_last_error()
    assert lib.tvl_attention_backward(attention_args(), grads_args(g_token=-64), P, 1 << 40, None) == 1 and b"stride" in lib.tvl_last_error()


def rotary_args(**kw):
    f = dict(size=A._ROTARY.size, x=P, y=P, positions=P, table=P, batch=2, tokens=3, heads=4, dim=64, rotary_dim=32, table_rows=16, ld_table=32,
             x_batch=0, x_token=0, x_head=0, y_batch=0, y_token=0, y_head=0, pos_batch=0, pos_token=0, dtype=1, interleaved=0, inverse=0, reserved=0)
    f.update(kw)
    return A._ROTARY.pack(*f.values())


def rotary_cache_args(**kw):
    f = dict(size=A._ROTARY_CACHE.size, qkv=P, q=P, k_cache=P, v_cache=P, table=P, cache_len=0, count=0, batch=2, tokens=3, heads=4, kv_heads=2, dim=64, rotary_dim=32,
             slots=8, table_rows=16, ld_table=32, x_batch=0, x_token=0, k_batch=0, k_head=0, k_slot=0, v_batch=0, v_head=0, v_slot=0,
             cache_len_stride=0, cache_len_value=0, dtype=1, interleaved=0)
    f.update(kw)
    return A._ROTARY_CACHE.pack(*f.values())


@pytest.mark.parametrize("kw", [dict(size=8), dict(dtype=4), dict(batch=-1), dict(rotary_dim=33), dict(rotary_dim=66), dict(ld_table=31), dict(tokens=1 << 31), dict(dim=1 << 13),
                                dict(table=0), dict(table=P + 2)])
def test_rotary_refusals(kw):
    assert lib.tvl_rotary(rotary_args(**kw), None) == 1
    assert lib.tvl_rotary_cache(rotary_cache_args(**kw), None) == 1


def test_rotary_refuses_null_pointers_and_skips_empty_calls():
    for name in ("x", "y", "positions"):
        assert lib.tvl_rotary(rotary_args(**{name: 0}), None) == 1 and b"NULL" in lib.tvl_last_error()
    for name in ("qkv", "q", "k_cache", "v_cache"):
        assert lib.tvl_rotary_cache(rotary_cache_args(**{name: 0}), None) == 1 and b"NULL" in lib.tvl_last_error()
    assert lib.tvl_rotary(None, None) == 1 and lib.tvl_rotary_cache(None, None) == 1
    for name in ("batch", "tokens", "dim"):
        kw = {name: 0, "rotary_dim": 0}
        assert lib.tvl_rotary(rotary_args(x=0, **kw), None) == 0 and lib.tvl_rotary_cache(rotary_cache_args(qkv=0, **kw), None) == 0


def test_cpu_tensors_are_refused():
    x = torch.zeros(1, 2, 4, 64)
    t = torch.zeros(8, 64)
    for call in (lambda: tv.rotary(x, torch.arange(2), t), lambda: tv.attention(x, x, x), lambda: tv.cached_attention(x, x, x, 0),
                 lambda: tv.rotary_cache(x.view(1, 2, 256), t, x, x.clone(), 0, 2)):
        with pytest.raises(ValueError, match="GPU"):
            call()
    with pytest.raises(TypeError):
        tv.attention([1.0], x, x)


def test_rotary_table():
    t = tv.rotary_table(8, 5, theta=100.0, device="cpu")
    assert t.shape == (5, 8) and t.dtype == torch.float32
    for p in range(5):
        for i in range(4):
            a = p * 100.0 ** (-2 * i / 8)
            # float64 angles, one rounding to float32
            assert abs(float(t[p, i]) - math.cos(a)) <= 2.0 ** -24 and abs(float(t[p, 4 + i]) - math.sin(a)) <= 2.0 ** -24
    far = tv.rotary_table(4, 200001, device="cpu")[200000]       # a far position keeps its digits
    assert abs(float(far[0]) - math.cos(200000.0)) <= 2.0 ** -24 and abs(float(far[3]) - math.sin(2000.0)) <= 2.0 ** -24
    lin = tv.rotary_table(8, 9, scaling="linear", factor=2.0, device="cpu")
    assert torch.equal(lin[::2], tv.rotary_table(8, 5, device="cpu"))
    ntk = tv.rotary_table(8, 2, scaling="ntk", factor=4.0, device="cpu")[1]
    assert abs(math.atan2(float(ntk[4]), float(ntk[0])) - 1.0) <= 1e-6                       # the fastest pair as before
    assert abs(math.atan2(float(ntk[7]), float(ntk[3])) - 10000.0 ** -0.75 / 4) <= 1e-8      # the slowest divided by the factor
    parts = tv.rotary_table(64, 2, scaling="parts", factor=8.0, original_len=2048, device="cpu")[1].double()
    amp = 0.1 * math.log(8.0) + 1.0
    for i in range(32):
        f = 10000.0 ** (-2 * i / 64)
        keep = min(1.0, max(0.0, (2048 * f / (2 * math.pi) - 1) / 31))
        f = f * keep + f / 8 * (1 - keep)
        assert abs(float(parts[i]) - amp * math.cos(f)) <= 2e-7 and abs(float(parts[32 + i]) - amp * math.sin(f)) <= 2e-7
    for bad in (dict(rotary_dim=3), dict(max_len=-1), dict(theta=0.0), dict(factor=0.5, scaling="linear"), dict(factor=2.0), dict(scaling="other"), dict(scaling="parts", factor=2.0),
                dict(rotary_dim=2, scaling="ntk", factor=2.0)):
        with pytest.raises(ValueError):
            tv.rotary_table(**{**dict(rotary_dim=8, max_len=4, device="cpu"), **bad})
    assert tv.rotary_table(0, 4, device="cpu").shape == (4, 0)
