"""Refusals of the 8-bit cache's entry points, and their workspace sizes:
arguments are checked before anything is launched, so no GPU is needed."""
import ctypes

import pytest
import torch

import canvas_attn as ca
from canvas_attn import kv8

FAKE = 1 << 40  # an aligned address nothing reads


def c_cache(**kw):
    d = dict(k=FAKE, v=FAKE, k_scale=FAKE, v_scale=FAKE, batch=2, n_total=100, n_head_kv=2,
             head_dim=128, block_tokens=32, row_stride=0)
    d.update(kw)
    return kv8.CaKv8Cache(**d)


BAD_CACHES = [
    (dict(k=None), ca.CA_ERR_INVALID), (dict(v_scale=None), ca.CA_ERR_INVALID),
    (dict(k=FAKE + 8), ca.CA_ERR_INVALID), (dict(batch=-1), ca.CA_ERR_INVALID),
    (dict(n_total=0), ca.CA_ERR_INVALID), (dict(n_head_kv=0), ca.CA_ERR_INVALID),
    (dict(head_dim=0), ca.CA_ERR_INVALID), (dict(head_dim=72), ca.CA_ERR_UNSUPPORTED),
    (dict(head_dim=528), ca.CA_ERR_UNSUPPORTED), (dict(block_tokens=48), ca.CA_ERR_UNSUPPORTED),
    (dict(block_tokens=0), ca.CA_ERR_UNSUPPORTED), (dict(row_stride=128), ca.CA_ERR_INVALID),
    (dict(row_stride=264), ca.CA_ERR_INVALID),
]


def store_call(cache=None, **kw):
    d = dict(k=FAKE, v=FAKE, n_active=4, active_pos=FAKE)
    d.update(kw)
    a = kv8.CaKv8StoreArgs(cache=cache or c_cache(), **d)
    return ca.lib.ca_kv8_store(ctypes.byref(a), None)


def load_call(cache=None, **kw):
    d = dict(pos=FAKE, n_pos=4, k_out=FAKE, v_out=FAKE)
    d.update(kw)
    a = kv8.CaKv8LoadArgs(cache=cache or c_cache(), **d)
    return ca.lib.ca_kv8_load(ctypes.byref(a), None)


def attn_args(cache=None, **kw):
    d = dict(q=FAKE, out=FAKE, n_head=4, sq=3, sliding_window=-1, causal_prefix=-1, scale=1.0)
    d.update(kw)
    return kv8.CaAttnKv8Args(cache=cache or c_cache(), **d)


def attn_call(cache=None, **kw):
    a = attn_args(cache, **kw)
    return ca.lib.ca_attention_kv8_dev(ctypes.byref(a), None)


@pytest.mark.parametrize("kw,status", BAD_CACHES)
def test_bad_caches_are_refused_everywhere(kw, status):
    for call in (store_call, load_call, attn_call):
        assert call(c_cache(**kw)) == status
    a = attn_args(c_cache(**kw))
    assert ca.lib.ca_attention_kv8_workspace(ctypes.byref(a)) == status


def test_null_arguments():
    for fn in (ca.lib.ca_kv8_store, ca.lib.ca_kv8_load, ca.lib.ca_attention_kv8_dev):
        assert fn(None, None) == ca.CA_ERR_INVALID
    assert ca.lib.ca_attention_kv8_workspace(None) == ca.CA_ERR_INVALID


@pytest.mark.parametrize("kw,status", [
    (dict(k=None), ca.CA_ERR_INVALID), (dict(v=FAKE + 2), ca.CA_ERR_INVALID),
    (dict(active_pos=None), ca.CA_ERR_INVALID), (dict(n_active=-1), ca.CA_ERR_INVALID),
    (dict(cu_active=FAKE, total_active=-1), ca.CA_ERR_INVALID),
    (dict(cu_active=FAKE, total_active=1 << 31), ca.CA_ERR_UNSUPPORTED),
    (dict(n_active=0), ca.CA_OK), (dict(cu_active=FAKE, total_active=0), ca.CA_OK),
])
def test_store_arguments(kw, status):
    assert store_call(**kw) == status


@pytest.mark.parametrize("kw,status", [
    (dict(k_out=None, v_out=None), ca.CA_ERR_INVALID), (dict(k_out=FAKE + 4), ca.CA_ERR_INVALID),
    (dict(n_pos=-1), ca.CA_ERR_INVALID), (dict(pos=None, n_pos=101), ca.CA_ERR_INVALID),
    (dict(n_pos=0), ca.CA_OK),
])
def test_load_arguments(kw, status):
    assert load_call(**kw) == status


@pytest.mark.parametrize("kw,status", [
    (dict(q=None), ca.CA_ERR_INVALID), (dict(out=None), ca.CA_ERR_INVALID),
    (dict(q=FAKE + 2), ca.CA_ERR_INVALID), (dict(out=FAKE + 8), ca.CA_ERR_INVALID),
    (dict(n_head=3), ca.CA_ERR_INVALID), (dict(n_head=0), ca.CA_ERR_INVALID),
    (dict(sq=-1), ca.CA_ERR_INVALID), (dict(cu_q=FAKE, max_sq=-1), ca.CA_ERR_INVALID),
    (dict(q_row_stride=500), ca.CA_ERR_INVALID), (dict(q_row_stride=516), ca.CA_ERR_INVALID),
    (dict(out_row_stride=514), ca.CA_ERR_INVALID),
    (dict(sq=0), ca.CA_OK), (dict(cu_q=FAKE, max_sq=0, total_q=0), ca.CA_OK),
])
def test_attention_arguments(kw, status):
    assert attn_call(**kw) == status


def test_caches_past_int32_rows_are_refused():
    big = c_cache(batch=2, n_total=(1 << 30) - 20)
    assert attn_call(big) == ca.CA_ERR_UNSUPPORTED


def block_call(cache=None, **kw):
    d = dict(q=FAKE, k=FAKE, v=FAKE, n_head=4, n_active=3, active_pos=FAKE, rope=FAKE, rope_len=100,
             rope_dim=128, work=FAKE, out=FAKE, sliding_window=-1, causal_prefix=-1, scale=1.0)
    d.update(kw)
    a = kv8.CaBlockKv8Args(cache=cache or c_cache(), **d)
    return ca.lib.ca_attention_block_kv8_dev(ctypes.byref(a), None)


@pytest.mark.parametrize("kw,status", [
    (dict(q=None), ca.CA_ERR_INVALID), (dict(work=None), ca.CA_ERR_INVALID),
    (dict(work=FAKE + 8), ca.CA_ERR_INVALID), (dict(active_pos=None), ca.CA_ERR_INVALID),
    (dict(rope_len=99), ca.CA_ERR_INVALID), (dict(rope_dim=130), ca.CA_ERR_INVALID),
    (dict(rope_dim=3), ca.CA_ERR_INVALID), (dict(n_head=3), ca.CA_ERR_INVALID),
    (dict(n_active=-1), ca.CA_ERR_INVALID), (dict(out=FAKE + 4), ca.CA_ERR_INVALID),
    (dict(cu_active=FAKE, total_active=3, max_active=-1), ca.CA_ERR_INVALID),
    (dict(out_row_stride=8), ca.CA_ERR_INVALID), (dict(n_active=0), ca.CA_OK),
])
def test_block_arguments(kw, status):
    assert block_call(**kw) == status


@pytest.mark.parametrize("kw,status", BAD_CACHES)
def test_block_refuses_bad_caches(kw, status):
    assert block_call(c_cache(**kw)) == status


def test_workspace_is_checked_and_sized():
    long = c_cache(batch=1, n_total=8192)
    a = attn_args(long, sq=1)
    n = kv8.workspace_bytes(a)
    assert n > kv8.TICKET_BYTES
    assert attn_call(long, sq=1, workspace=FAKE, workspace_bytes=n - 1) == ca.CA_ERR_INVALID
    assert attn_call(long, sq=1, workspace=FAKE + 4, workspace_bytes=n) == ca.CA_ERR_INVALID
    # Short or many key axes are not split and need none.
    assert kv8.workspace_bytes(attn_args(c_cache(batch=1), sq=1)) == 0
    assert kv8.workspace_bytes(attn_args(c_cache(batch=512, n_total=8192), sq=1)) == 0


def test_python_checks():
    cache = kv8.Kv8Cache.alloc(2, 40, 2, 64, block_tokens=16, device="cpu")
    assert cache.k_scale.shape == (2, 3, 2)
    bf = torch.bfloat16
    x = torch.zeros(2, 3, 2, 64, dtype=bf)
    pos = torch.zeros(2, 3, dtype=torch.int32)
    kv8.make_store_args(cache, x, x, pos)
    for bad in (dict(k=x.float()), dict(v=x[:, :2]), dict(active_pos=pos.long()),
                dict(active_pos=pos[:1]), dict(k=x.transpose(0, 1)), dict(kv_len=pos)):
        kw = dict(k=x, v=x, active_pos=pos)
        kw.update(bad)
        with pytest.raises(ValueError):
            kv8.make_store_args(cache, **kw)
    q = torch.zeros(2, 3, 4, 64, dtype=bf)
    kv8.make_attention_args(q, cache, q.clone(), q_pos=pos, workspace=False)
    for bad in (dict(q=q.float()), dict(out=q.double()), dict(q_pos=pos.long()),
                dict(q=q[:1], out=q[:1]), dict(out=q.transpose(2, 3)), dict(kv_len=pos)):
        kw = dict(q=q, out=q.clone(), q_pos=pos, workspace=False)
        kw.update(bad)
        with pytest.raises(ValueError):
            kv8.make_attention_args(cache=cache, **kw)
    with pytest.raises(ValueError):
        kv8.make_load_args(cache, None, None)
    with pytest.raises(ValueError):
        kv8.make_load_args(cache, x, x.float())
    with pytest.raises(ValueError):
        kv8.Kv8Cache(cache.k, cache.v[:, :30], cache.k_scale, cache.v_scale, 16).to_c()
    with pytest.raises(ValueError):
        kv8.Kv8Cache(cache.k, cache.v, cache.k_scale, cache.v_scale, 32).to_c()
    with pytest.raises(ValueError):
        kv8.Kv8Cache(cache.k, cache.v, cache.k_scale, cache.v_scale, 24).to_c()


def test_ragged_rows_need_their_largest_count():
    # With the count left at 0, or too small for the rows, rows would be left
    # unwritten: refused by the C entries before anything is launched ...
    ragged = dict(cu_q=FAKE, total_q=9)
    for max_sq, status in ((0, ca.CA_ERR_INVALID), (4, ca.CA_ERR_INVALID)):
        assert attn_call(max_sq=max_sq, **ragged) == status
        a = attn_args(max_sq=max_sq, **ragged)
        assert ca.lib.ca_attention_kv8_workspace(ctypes.byref(a)) == status
        assert block_call(cu_active=FAKE, total_active=9, max_active=max_sq) == status
    assert kv8.workspace_bytes(attn_args(max_sq=5, **ragged)) >= 0
    # ... and by Python, where it has a default.
    cache = kv8.Kv8Cache.alloc(2, 40, 2, 64, block_tokens=16, device="cpu")
    q = torch.zeros(3, 4, 64, dtype=torch.bfloat16)
    kv = torch.zeros(3, 2, 64, dtype=torch.bfloat16)
    cu = torch.tensor([0, 1, 3], dtype=torch.int32)
    kv8.make_attention_args(q, cache, q.clone(), cu_q=cu, max_sq=2, workspace=False)
    for kw in (dict(), dict(max_sq=1)):
        with pytest.raises(ValueError, match="max_sq"):
            kv8.make_attention_args(q, cache, q.clone(), cu_q=cu, workspace=False, **kw)
    block = dict(active_pos=torch.zeros(3, dtype=torch.int32), rope=torch.zeros(40, 2), rope_len=40,
                 rope_dim=0, cu_active=cu, workspace=False)
    kv8.make_block_args(q, kv, kv, cache, q.clone(), max_active=2, **block)
    for kw in (dict(), dict(max_active=1)):
        with pytest.raises(ValueError, match="max_active"):
            kv8.make_block_args(q, kv, kv, cache, q.clone(), **kw, **block)


@pytest.mark.parametrize("batch,n,stride", [(3, 5, 256), (3, 1, 256), (1, 5, 256), (1, 1, 0)])
def test_stride_of_a_cache_in_wider_rows(batch, n, stride):
    # The first 2 of 4 heads; with one position a sequence the stride is still
    # what lies between the sequences.
    wide = kv8.Kv8Cache.alloc(batch, n, 4, 64, block_tokens=16, device="cpu")
    cut = kv8.Kv8Cache(wide.k[:, :, :2], wide.v[:, :, :2], wide.k_scale[:, :, :2].contiguous(),
                       wide.v_scale[:, :, :2].contiguous(), 16)
    assert cut.to_c().row_stride == stride
