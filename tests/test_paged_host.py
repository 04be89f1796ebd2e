"""The paged-cache entry points' refusals and the rotary plans: no GPU needed."""
import ctypes

import pytest

from anedvd_b200 import runtime as rt

A = 0x10000  # an aligned address that no refused call reads


def kv(**k):
    return rt.CuqPagedKv(**{**dict(k=A, v=A, type=1, n_pages=8, page_size=16, kv_heads=2, head_dim=64, page_stride=0), **k})


def batch(**k):
    return rt.CuqBatch(**{**dict(q_start=A, kv_len=A, pages=A, n_seqs=2, n_tok=4, pages_stride=4, max_q=2, max_kv=64), **k})


BAD_KV = [(dict(type=0), rt.EUNSUPPORTED), (dict(type=8), rt.EUNSUPPORTED), (dict(head_dim=96), rt.EUNSUPPORTED),
          (dict(page_size=8), rt.EUNSUPPORTED), (dict(page_size=48), rt.EUNSUPPORTED), (dict(page_size=512), rt.EUNSUPPORTED),
          (dict(k=None), rt.EINVAL), (dict(v=A + 8), rt.EINVAL), (dict(kv_heads=0), rt.EINVAL), (dict(n_pages=0), rt.EINVAL),
          (dict(page_stride=2047), rt.EINVAL), (dict(page_stride=2052), rt.EINVAL)]
BAD_BATCH = [(dict(kv_len=None), rt.EINVAL), (dict(pages=A + 2), rt.EINVAL), (dict(n_seqs=70000), rt.EINVAL),
             (dict(n_tok=1 << 30), rt.EINVAL), (dict(max_kv=1 << 31), rt.EINVAL)]



def append(c=None, b=None, rot=64, **k):
    a = dict(positions=None, q_out=A, q_out_stride=256, out_type=1, q=A + 64, q_stride=512, k=A, v=A, kv_stride=512,
             in_type=1, heads=4)
    a.update(k)
    p = rt.RopePlan(rt.CuqRopeParams(rot_dim=rot, theta=1e4))
    return rt.load().cuq_rope_append(p.handle, ctypes.byref(c or kv()), ctypes.byref(b or batch()), *a.values(), None)


def attention(c=None, b=None, **k):
    a = dict(out=A, out_stride=256, q=A + 64, q_stride=256, type=1, lse=A, heads=4, scale=0.1, causal=1, window=0,
             workspace=A, bytes=1 << 40)
    a.update(k)
    return rt.load().cuq_attention_paged(ctypes.byref(c or kv()), ctypes.byref(b or batch()), *a.values(), None)


def mass(c=None, b=None, **k):
    a = dict(mass=A, stride=64, q=A, q_stride=256, type=1, lse=A, heads=4, scale=0.1, causal=1, window=0, last_q=0,
             decay=1.0)
    a.update(k)
    return rt.load().cuq_attention_mass(ctypes.byref(c or kv()), ctypes.byref(b or batch()), *a.values(), None)


def evict(c=None, b=None, **k):
    a = dict(mass=A, stride=64, keep=8, sink=2, recent=2, kept=A, new_len=A + 64, mass_out=None, out_stride=64)
    a.update(k)
    return rt.load().cuq_kv_evict(ctypes.byref(c or kv()), ctypes.byref(b or batch()), *a.values(), None)


@pytest.mark.parametrize("call", [append, attention, mass, evict])
@pytest.mark.parametrize("bad,code", BAD_KV)
def test_bad_caches_are_refused(call, bad, code):
    assert call(c=kv(**bad)) == code
    assert rt.last_error()


@pytest.mark.parametrize("call", [append, attention, mass, evict])
@pytest.mark.parametrize("bad,code", BAD_BATCH)
def test_bad_batches_are_refused(call, bad, code):
    assert call(b=batch(**bad)) == code


@pytest.mark.parametrize("call", [append, attention, mass])
def test_query_ops_need_q_start_and_whole_groups(call):
    assert call(b=batch(q_start=None)) == rt.EINVAL
    assert call(heads=5) == rt.EINVAL
    assert call(heads=0) == rt.EINVAL


@pytest.mark.parametrize("bad,code", [
    (dict(in_type=8), rt.EUNSUPPORTED), (dict(out_type=30), rt.EUNSUPPORTED), (dict(rot=128), rt.EINVAL),
    (dict(q=A + 4), rt.EINVAL), (dict(k=None), rt.EINVAL), (dict(q_stride=255), rt.EINVAL), (dict(q_stride=252), rt.EINVAL),
    (dict(kv_stride=120), rt.EINVAL), (dict(q_out_stride=248), rt.EINVAL), (dict(positions=A + 1), rt.EINVAL),
    (dict(q_out=A + 64, q_stride=512, q_out_stride=256), rt.EINVAL)])
def test_append_refusals(bad, code):
    assert append(**bad) == code


@pytest.mark.parametrize("bad,code", [
    (dict(type=30), rt.EUNSUPPORTED), (dict(type=8), rt.EUNSUPPORTED), (dict(q=None), rt.EINVAL), (dict(q=A + 8), rt.EINVAL),
    (dict(q_stride=248), rt.EINVAL), (dict(scale=float("nan")), rt.EINVAL), (dict(scale=float("inf")), rt.EINVAL),
    (dict(causal=0, window=5), rt.EINVAL)])
@pytest.mark.parametrize("call", [attention, mass])
def test_query_refusals(call, bad, code):
    assert call(**bad) == code


def test_fp32_queries_need_an_fp16_cache():
    assert attention(c=kv(type=30), type=0) == rt.EUNSUPPORTED
    assert mass(c=kv(type=30), type=0) == rt.EUNSUPPORTED


def test_attention_refusals():
    assert attention(out=A + 64) == rt.EINVAL          # out is q
    assert attention(out=A + 4) == rt.EINVAL
    assert attention(out_stride=252) == rt.EINVAL
    assert attention(lse=A + 2) == rt.EINVAL
    b = batch(n_seqs=1, max_q=1, max_kv=100000, pages_stride=6250)
    need = rt.load().cuq_attention_paged_workspace(ctypes.byref(kv()), ctypes.byref(b), 4, 1)
    if need:
        assert attention(b=b, bytes=need - 1) == rt.EINVAL
        assert attention(b=b, workspace=None) == rt.EINVAL
        assert attention(b=b, workspace=A + 16) == rt.EINVAL


def test_mass_and_evict_refusals():
    assert mass(stride=63) == rt.EINVAL
    assert mass(mass=None) == rt.EINVAL and mass(lse=None) == rt.EINVAL
    assert mass(decay=float("nan")) == rt.EINVAL
    assert evict(keep=0) == rt.EINVAL
    assert evict(keep=3) == rt.EINVAL                  # sink + recent
    assert evict(sink=0xFFFFFFFF, recent=9) == rt.EINVAL
    assert evict(stride=63) == rt.EINVAL
    assert evict(new_len=A) == rt.EINVAL               # the batch's kv_len
    assert evict(kept=None) == rt.EINVAL
    assert evict(mass_out=A + 4, out_stride=63) == rt.EINVAL
    assert evict(mass_out=A, stride=64, out_stride=80) == rt.EINVAL


def test_empty_batches_are_no_work():
    assert append(b=batch(n_seqs=0)) == rt.OK
    assert append(b=batch(n_tok=0)) == rt.OK
    assert attention(b=batch(n_seqs=0)) == rt.OK
    assert attention(b=batch(max_q=0)) == rt.OK
    assert mass(b=batch(n_seqs=0)) == rt.OK
    assert mass(b=batch(max_kv=0)) == rt.OK
    assert evict(b=batch(n_seqs=0)) == rt.OK


@pytest.mark.parametrize("bad", [
    dict(rot_dim=0), dict(rot_dim=24), dict(rot_dim=144), dict(theta=1.0), dict(theta=float("nan")), dict(scaling=4),
    dict(scaling=-1), dict(scaling=1, factor=0.5), dict(scaling=2, factor=8.0), dict(scaling=3, factor=4.0),
    dict(scaling=2, factor=8.0, orig_ctx=8192, low_freq=4.0, high_freq=1.0),
    dict(scaling=3, factor=4.0, orig_ctx=4096, beta_fast=1.0, beta_slow=32.0),
    dict(scaling=3, factor=4.0, orig_ctx=4096, beta_fast=32.0, beta_slow=1.0, attn_factor=-1.0)])
def test_rope_plans_are_checked(bad):
    with pytest.raises(rt.CuqError):
        rt.RopePlan(rt.CuqRopeParams(**{**dict(rot_dim=64, theta=1e4), **bad}))


def test_null_descriptors():
    L = rt.load()
    assert L.cuq_rope_append(None, None, None, *([None] * 2), 0, 0, None, 0, None, None, 0, 0, 0, None) == rt.EINVAL
    assert L.cuq_attention_paged(None, None, None, 0, None, 0, 0, None, 0, 0.0, 0, 0, None, 0, None) == rt.EINVAL
    assert L.cuq_attention_mass(None, None, None, 0, None, 0, 0, None, 0, 0.0, 0, 0, 0, 0.0, None) == rt.EINVAL
    assert L.cuq_kv_evict(None, None, None, 0, 0, 0, 0, None, None, None, 0, None) == rt.EINVAL
    assert L.cuq_attention_paged_workspace(None, None, 0, 0) == 0
