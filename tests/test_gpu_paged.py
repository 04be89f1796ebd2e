"""The paged-cache ops against a 64-bit model of their definitions, at the sizes and masks where they can go wrong.

Tolerances count roundings.  Rotation: two products, a sum, and a cosine and sine off by at most 2^-22 (2 ulp of 1 and
pi 2^-25 from the fp32 turn): 2^-21 (|a| + |b|), then half a step of the output.  Attention over fp16 / bf16: each
probability is rounded once (u of itself, twice where the sum is of the unrounded ones) and the output once; fp32 score
sums of 128 products are off by at most 2^-17 of sum |q k|, which moves a probability by twice that.  fp32 queries: the
dropped low parts are 2^-22 of sum |q k| (inside the same 2^-17), probabilities split in two fp16 are off by 2^-21 of
themselves and by at most 2^-25 of the largest where the low part is subnormal.
"""
import ctypes
import math

import pytest
import torch

from anedvd_b200 import runtime as rt

from . import paged_util as pu
from .gpu_util import lib, ptr

pytestmark = pytest.mark.gpu

PAIRS = [("f32", "f16"), ("f16", "f16"), ("bf16", "bf16")]


def queries(b, heads, t, seed=1, pad=0):
    """q [n_tok][heads][hd] as a view of rows `pad` wider, and its row stride."""
    g = torch.Generator().manual_seed(seed)
    row = heads * b.hd + pad
    base = (1.5 * torch.randn(max(1, b.n_tok), row, generator=g)).to(pu.DT[t]).cuda()
    return base, row, base[: b.n_tok, : heads * b.hd].reshape(b.n_tok, heads, b.hd).cpu()


def attend(b, heads, t, q, q_row, scale, causal=True, window=0, out_pad=0, fill=7.0, stream=None, lse=True):
    L = lib()
    row = heads * b.hd + out_pad
    out = torch.full((max(1, b.n_tok), row), fill, dtype=pu.DT[t], device="cuda")
    ls = torch.full((max(1, b.n_tok), heads), fill, dtype=torch.float32, device="cuda")
    need = L.cuq_attention_paged_workspace(b.kvp, b.bp, heads, pu.GGML[t])
    ws = torch.full((max(1, need),), 255, dtype=torch.uint8, device="cuda")  # whatever it holds
    rt.check(L.cuq_attention_paged(b.kvp, b.bp, ptr(out), row, ptr(q), q_row, pu.GGML[t], ptr(ls) if lse else None,
                                   heads, scale, int(causal), window, ptr(ws), need, stream))
    rt.check(L.cuq_paged_status(stream))
    return out, ls


def check_attention(b, heads, t, got, lse, q_host, scale, causal=True, window=0, fill=7.0):
    want, wl, mag, top = b.attention(q_host, scale, causal, window)
    o = got[: b.n_tok, : heads * b.hd].reshape(b.n_tok, heads, b.hd).double().cpu()
    u, used = pu.unit(t), b.used
    d = 2 * top[..., None] * 2.0 ** -17
    if t == "f32":
        n = max([x for _, x in b.seqs] + [1])
        vmax = float(b.v_host.double().abs().max())
        tol = mag * (d + 2.0 ** -19) + 2.0 ** -24 * want.abs() + n * 2.0 ** -25 * vmax + 1e-30
    else:
        tol = mag * (2 * u + d + 2.0 ** -19) + 1.01 * u * want.abs() + 2.0 ** -25
    bad = (o[:used] - want[:used]).abs() - tol[:used]
    assert not o[:used].isnan().any()
    assert bad.numel() == 0 or float(bad.max()) <= 0, float(bad.max())
    assert (o[used:] == fill).all()                                            # rows of no sequence
    assert (got[: b.n_tok, heads * b.hd:] == fill).all()                       # and the padding of each row
    l = lse[: b.n_tok].double().cpu()
    empty = wl[:used].isinf()
    assert (l[:used][empty] == -math.inf).all() and (o[:used][empty] == 0).all()
    ltol = (2.0 ** -17 * top + 2.0 ** -20 * (1 + wl.abs()))[:used][~empty]
    assert ((l[:used] - wl[:used])[~empty].abs() <= ltol).all()
    assert (l[used:] == fill).all()


def run_attention(seqs, heads, kv_heads, hd, pair, page=16, causal=True, window=0, holes=(), tail=0, page_pad=0,
                  q_pad=0, out_pad=0, seed=0):
    t, cache = pair
    b = pu.Batch(seqs, kv_heads, hd, cache, page, seed, tail, holes, page_pad)
    q, row, qh = queries(b, heads, t, seed + 1, q_pad)
    scale = hd ** -0.5
    out, lse = attend(b, heads, t, q, row, scale, causal, window, out_pad)
    check_attention(b, heads, t, out, lse, qh, scale, causal, window)
    assert torch.equal(b.k.cpu(), b.k_host) and torch.equal(b.v.cpu(), b.v_host)


TOKENS = [(1, n) for n in (1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 128, 129, 255, 257, 1000, 2500)]
GEOS = [(9, 3, 64), (14, 2, 64), (12, 2, 128), (32, 8, 128), (8, 8, 64), (8, 1, 128), (20, 1, 64)]


@pytest.mark.parametrize("geo", GEOS)
@pytest.mark.parametrize("pair", PAIRS)
def test_single_tokens_of_every_length(geo, pair):
    run_attention(TOKENS, *geo, pair)


def workspace_of(seqs, heads, kv_heads, hd, pair):
    b = pu.Batch(seqs, kv_heads, hd, pair[1])
    return lib().cuq_attention_paged_workspace(b.kvp, b.bp, heads, pu.GGML[pair[0]])


@pytest.mark.parametrize("geo", GEOS)
@pytest.mark.parametrize("pair", PAIRS)
@pytest.mark.parametrize("n", [1, 16, 40, 200, 609, 1100, 2000, 4000])
def test_one_token_of_one_sequence(n, pair, geo):
    """Short caches: a cluster of 1 to 8 CTAs joins its own parts, without a workspace (up to 16 heads a KV head)."""
    assert workspace_of([(1, n)], *geo, pair) == 0 or geo[0] // geo[1] > 16
    run_attention([(1, n)], *geo, pair, seed=n)


@pytest.mark.parametrize("geo", GEOS)
@pytest.mark.parametrize("pair", PAIRS)
def test_short_caches(geo, pair):
    """Ragged ones, an empty cache, a sequence without tokens, rows behind the last sequence."""
    seqs = [(1, 1), (1, 17), (0, 40), (1, 129), (1, 0), (1, 33), (1, 480), (1, 16), (1, 255), (0, 0), (1, 500)]
    assert workspace_of(seqs, *geo, pair) == 0 or geo[0] // geo[1] > 16
    run_attention(seqs, *geo, pair, tail=3, q_pad=8, out_pad=16, page_pad=64, seed=11)


@pytest.mark.parametrize("geo", [(8, 8, 64), (4, 1, 128), (14, 2, 64)])
@pytest.mark.parametrize("pair", PAIRS)
@pytest.mark.parametrize("window", [0, 1, 40, 300])
def test_short_drafts(window, pair, geo):
    """As many tokens as one tile of 16 rows holds, through windows, holes and a mask that is not causal."""
    q = 16 * geo[1] // geo[0]
    seqs = [(q, 900), (1, 333), (q, q), (q, max(0, q - 2)), (q, 64)]
    assert workspace_of(seqs, *geo, pair) == 0
    holes = [(0, 0), (0, 3), (0, 55), (0, 56), (1, 20), (4, 0), (4, 1), (4, 2), (4, 3)]
    run_attention(seqs, *geo, pair, window=window, holes=holes, seed=window + 13)
    if not window:
        run_attention(seqs, *geo, pair, causal=False, holes=holes, seed=17)


@pytest.mark.parametrize("geo", [(9, 3, 64), (32, 8, 128)])
@pytest.mark.parametrize("pair", PAIRS)
def test_short_and_long_bounds_agree(geo, pair):
    """The same caches under a bound that asks for runs and the merge: equal within both paths' roundings."""
    heads, kv_heads, hd = geo
    t, cache = pair
    b = pu.Batch([(1, 700), (1, 20), (1, 413)], kv_heads, hd, cache, seed=23)
    q, row, qh = queries(b, heads, t, 24)
    near = attend(b, heads, t, q, row, hd ** -0.5)
    check_attention(b, heads, t, *near, qh, hd ** -0.5)
    wide = torch.full((3, 1024), -1, dtype=torch.int32)
    wide[:, : b.table.shape[1]] = b.table
    b.d_wide = wide.cuda()
    b.desc.pages, b.desc.pages_stride, b.desc.max_kv = b.d_wide.data_ptr(), 1024, 16384
    assert lib().cuq_attention_paged_workspace(b.kvp, b.bp, heads, pu.GGML[t]) > 0
    far = attend(b, heads, t, q, row, hd ** -0.5)
    check_attention(b, heads, t, *far, qh, hd ** -0.5)


@pytest.mark.parametrize("pair", PAIRS)
@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
def test_page_sizes(page, pair):
    run_attention([(1, 777), (5, 300), (70, 513), (1, page), (3, page + 1)], 12, 2, 128, pair, page=page)
    run_attention([(1, 777), (5, 300), (70, 513), (1, page), (3, page + 1)], 9, 3, 64, pair, page=page)


@pytest.mark.parametrize("geo", GEOS)
@pytest.mark.parametrize("pair", PAIRS)
def test_chunks(geo, pair):
    run_attention([(2, 2), (5, 40), (16, 17), (33, 33), (128, 300), (129, 129), (1, 77), (200, 1001)], *geo, pair,
                  tail=3, seed=3)


@pytest.mark.parametrize("pair", PAIRS)
@pytest.mark.parametrize("hd", [64, 128])
def test_long_chunk(pair, hd):
    run_attention([(700, 1500)], 4, 2, hd, pair, page=64, seed=5)


@pytest.mark.parametrize("pair", PAIRS)
def test_long_context(pair):
    run_attention([(1, 20011), (3, 9000)], 8, 2, 128, pair, page=32, seed=6)
    run_attention([(40, 12000)], 8, 2, 64, pair, page=16, seed=6)


@pytest.mark.parametrize("pair", PAIRS)
def test_rows_that_see_nothing(pair):
    # more new tokens than slots, no slots, no tokens, a sequence of holes only
    run_attention([(5, 3), (4, 0), (0, 9), (0, 0), (140, 20), (2, 40)], 6, 2, 64, pair,
                  holes=[(5, 0), (5, 1), (5, 2)], tail=2)
    run_attention([(0, 0), (0, 5)], 6, 2, 64, pair, tail=4)


@pytest.mark.parametrize("pair", PAIRS)
@pytest.mark.parametrize("window", [1, 7, 16, 100, 5000])
def test_windows_and_holes(window, pair):
    # pages behind the window are holes, and some inside it are too
    run_attention([(1, 900), (40, 500), (150, 400), (6, 5)], 12, 2, 128, pair, page=32, window=window,
                  holes=[(0, 0), (0, 1), (1, 3), (2, 0), (2, 11), (0, 28)], tail=1, seed=7)


@pytest.mark.parametrize("pair", PAIRS)
def test_not_causal(pair):
    run_attention([(1, 300), (9, 300), (130, 257), (8, 3), (300, 0)], 14, 2, 64, pair, causal=False, holes=[(1, 4)])


@pytest.mark.parametrize("pair", PAIRS)
def test_strides(pair):
    run_attention([(1, 50), (20, 70), (150, 200)], 6, 3, 128, pair, page_pad=24, q_pad=40, out_pad=8, tail=2)


@pytest.mark.parametrize("pair", PAIRS)
def test_extreme_scores(pair):
    """Scores of hundreds, and masked slots that hold infinities and NaN."""
    t, cache = pair
    b = pu.Batch([(1, 130), (20, 61), (150, 150)], 2, 64, cache, 32)
    g = torch.Generator().manual_seed(9)
    for pool, dev in ((b.k_host, b.k), (b.v_host, b.v)):
        pool.mul_(4.0)
        dev.copy_(pool)
        for i, (_, n) in enumerate(b.seqs):                # slots past each sequence's end
            page = int(b.table[i, n // 32]) if n % 32 else -1
            if page >= 0:
                p = dev.view(b.n_pages, 2, 32, 64)
                p[page, :, n % 32:] = float([math.nan, math.inf, -math.inf][i])
    q = (30 * torch.randn(b.n_tok, 4, 64, generator=g)).to(pu.DT[t])
    out, lse = attend(b, 4, t, q.cuda(), 256, 0.125)
    check_attention(b, 4, t, out, lse, q, 0.125)


def test_lse_is_optional_and_runs_repeat():
    b = pu.Batch([(1, 700), (30, 90), (200, 300)], 2, 128, "bf16")
    q, row, _ = queries(b, 8, "bf16")
    a, _ = attend(b, 8, "bf16", q, row, 0.1)
    c, l = attend(b, 8, "bf16", q, row, 0.1, lse=False)
    assert torch.equal(a, c) and (l == 7).all()


def test_max_bounds_cut():
    """Lengths past max_kv are cut, tokens past max_q are left as they are."""
    b = pu.Batch([(3, 100), (9, 80)], 2, 64, "f16")
    q, row, qh = queries(b, 4, "f16")
    b.desc.max_q = 3
    out, _ = attend(b, 4, "f16", q, row, 0.125)
    full = pu.Batch([(3, 100), (9, 80)], 2, 64, "f16")
    want, _, _, _ = full.attention(qh, 0.125)
    o = out[: b.n_tok].view(b.n_tok, 4, 64).double().cpu()
    assert (o[6:] == 7).all() and ((o[:6] - want[:6]).abs() < 0.01).all()
    b.desc.max_q, b.desc.max_kv = 9, 80
    out, _ = attend(b, 4, "f16", q, row, 0.125)
    cut = pu.Batch([(3, 100), (9, 80)], 2, 64, "f16")
    cut.seqs[0] = (3, 80)
    want, _, _, _ = cut.attention(qh, 0.125)
    o = out[: b.n_tok].view(b.n_tok, 4, 64).double().cpu()
    assert ((o - want).abs() < 0.01).all()


def test_bad_batch_arrays_touch_nothing():
    """q_start that falls, goes below zero or past n_tok, and negative lengths: cut, never out of bounds."""
    b = pu.Batch([(4, 50), (4, 50), (4, 50)], 2, 64, "f16")
    q, row, _ = queries(b, 4, "f16")
    for starts, lens in (([0, 9, 3, 12], [50, 50, 50]), ([-5, 2, 900, 1 << 30], [50, -7, 1 << 30]),
                         ([0, 4, 8, 12], [1 << 30, -(1 << 31), 50])):
        b.d_start.copy_(torch.tensor(starts, dtype=torch.int32))
        b.d_len.copy_(torch.tensor(lens, dtype=torch.int32))
        out, lse = attend(b, 4, "f16", q, row, 0.125)
        assert not out.isnan().any()


@pytest.mark.parametrize("pair", PAIRS)
def test_wide_groups(pair):
    """More query heads a KV head than a tile has rows."""
    run_attention([(1, 40), (3, 130), (2, 2)], 300, 1, 64, pair, page=32)
    run_attention([(1, 300), (5, 77)], 17, 1, 128, pair, page=32)


@pytest.mark.parametrize("pair", PAIRS)
def test_many_sequences(pair):
    """Hundreds of sequences: single tokens alone, and mixed with chunks and empty ones."""
    run_attention([(1, 1 + (37 * i) % 90) for i in range(1100)], 4, 2, 64, pair, tail=1)
    run_attention([((0, 1, 1, 9, 1)[i % 5], (i * 29) % 120 if i % 5 else 40) for i in range(300)], 6, 2, 64, pair, window=50)


@pytest.mark.parametrize("scale", [-0.2, 0.0, 1e-3])
def test_scales(scale):
    for pair in PAIRS:
        t, cache = pair
        b = pu.Batch([(1, 70), (40, 90), (150, 150)], 2, 64, cache, 16)
        q, row, qh = queries(b, 4, t)
        out, lse = attend(b, 4, t, q, row, scale)
        check_attention(b, 4, t, out, lse, qh, scale)


def test_offsets_past_32_bits():
    """Pools of more than 2^32 elements, with the pages at their far end."""
    stride, n_pages = 1 << 28, 18                       # 4.8e9 elements, 9.7 GB a pool
    b = pu.Batch([(1, 70), (33, 60)], 1, 64, "f16", 16)
    far = {n: torch.empty(n_pages, stride, dtype=torch.float16, device="cuda") for n in ("k", "v")}
    ids = list(range(n_pages - b.n_pages, n_pages)) if b.n_pages <= n_pages else None
    assert ids
    for i, p in enumerate(ids):
        far["k"][p, : b.stride] = b.k[i]
        far["v"][p, : b.stride] = b.v[i]
    b.table = torch.where(b.table < b.n_pages, b.table + ids[0], torch.tensor(1 << 30, dtype=torch.int32))
    b.d_table.copy_(b.table)
    near_k, near_v, first = b.k_host, b.v_host, ids[0]
    b.kv_desc.k, b.kv_desc.v = far["k"].data_ptr(), far["v"].data_ptr()
    b.kv_desc.page_stride, b.kv_desc.n_pages = stride, n_pages
    L = lib()
    row = (4 + 2) * 64
    x = torch.randn(b.n_tok, row, device="cuda").half()
    q = torch.empty(b.n_tok, 4 * 64, dtype=torch.float16, device="cuda")
    plan = rt.RopePlan(rt.CuqRopeParams(rot_dim=64, theta=1e4))
    rt.check(L.cuq_rope_append(plan.handle, b.kvp, b.bp, None, ptr(q), 256, 1, ptr(x), row,
                               ctypes.c_void_p(x.data_ptr() + 512), ctypes.c_void_p(x.data_ptr() + 640), row, 1, 4, None))
    out, lse = attend(b, 4, "f16", q, 256, 0.125)
    mass = torch.zeros(2, 1, b.max_kv, device="cuda")
    rt.check(L.cuq_attention_mass(b.kvp, b.bp, ptr(mass), b.max_kv, ptr(q), 256, 1, ptr(lse), 4, 0.125, 1, 0, 0, 1.0, None))
    rt.check(L.cuq_paged_status(None))
    # the model sees the same rows in small pools
    b.k_host = torch.stack([far["k"][p, : b.stride].cpu() for p in ids])
    b.v_host = torch.stack([far["v"][p, : b.stride].cpu() for p in ids])
    assert not torch.equal(b.k_host, near_k) and not torch.equal(b.v_host, near_v)
    b.table = torch.where(b.table < n_pages, b.table - first, b.table)
    check_attention(b, 4, "f16", out, lse, q.view(b.n_tok, 4, 64).cpu(), 0.125)
    for i, (_, n) in enumerate(b.seqs):
        want = 4.0 * b.seqs[i][0]
        assert abs(float(mass[i, :, :n].sum()) - want) < 2.0 ** -10 * want
    m0 = mass.cpu()
    kept = torch.empty(2, 1, 20, dtype=torch.int32, device="cuda")
    new = torch.empty(2, dtype=torch.int32, device="cuda")
    rt.check(L.cuq_kv_evict(b.kvp, b.bp, ptr(mass), b.max_kv, 20, 2, 4, ptr(kept), ptr(new), None, b.max_kv, None))
    torch.cuda.synchronize()
    for i, (_, n) in enumerate(b.seqs):
        keep = pu.evict(m0[i, 0], n, 20, 2, 4)
        assert kept[i, 0].tolist() == keep
        rows, _ = b.rows(b.k_host, i, n)
        for j, s in enumerate(keep):
            page = int(b.table[i, j // 16]) + first
            assert torch.equal(far["k"][page, (j % 16) * 64:(j % 16 + 1) * 64].cpu().double(), rows[s, 0])


def test_captured_before_any_other_call():
    """A process whose first call of each op is made while a graph is captured."""
    import subprocess
    import sys

    code = """
import ctypes, torch
from tests import paged_util as pu
from tests.test_gpu_paged import *
L = rt.load(); rt.init(0)
b = pu.Batch([(1, 40), (40, 300), (1, 7)], 2, 128, "bf16", 16)
q, row, qh = queries(b, 8, "bf16")
need = L.cuq_attention_paged_workspace(b.kvp, b.bp, 8, 30)
ws = torch.empty(max(1, need), dtype=torch.uint8, device="cuda")
out, lse = torch.full((b.n_tok, 1024), 7.0, dtype=torch.bfloat16, device="cuda"), torch.full((b.n_tok, 8), 7.0, device="cuda")
mass = torch.zeros(3, 2, b.max_kv, device="cuda")
kept = torch.empty(3, 2, 30, dtype=torch.int32, device="cuda"); new = torch.empty(3, dtype=torch.int32, device="cuda")
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    s = torch.cuda.current_stream().cuda_stream
    rt.check(L.cuq_attention_paged(b.kvp, b.bp, ptr(out), 1024, ptr(q), row, 30, ptr(lse), 8, 0.1, 1, 0, ptr(ws), need, s))
    rt.check(L.cuq_attention_mass(b.kvp, b.bp, ptr(mass), b.max_kv, ptr(q), row, 30, ptr(lse), 8, 0.1, 1, 0, 0, 1.0, s))
    rt.check(L.cuq_kv_evict(b.kvp, b.bp, ptr(mass), b.max_kv, 30, 2, 4, ptr(kept), ptr(new), None, b.max_kv, s))
g.replay(); torch.cuda.synchronize()
check_attention(b, 8, "bf16", out, lse, qh, 0.1)
assert new.tolist() == [30, 30, 7]
print("captured")
"""
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=240)
    assert "captured" in r.stdout, r.stdout[-2000:] + r.stderr[-2000:]


# ------------------------------------------------------------------ rotary + append ----

ROPES = [dict(rot_dim=64), dict(rot_dim=64, adjacent=1, theta=5e5), dict(rot_dim=32, scaling=rt.ROPE_LINEAR, factor=4.0),
         dict(rot_dim=16, adjacent=1, scaling=rt.ROPE_LLAMA3, factor=8.0, low_freq=1.0, high_freq=4.0, orig_ctx=8192),
         dict(rot_dim=64, scaling=rt.ROPE_YARN, factor=4.0, beta_fast=32.0, beta_slow=1.0, orig_ctx=4096),
         dict(rot_dim=48, scaling=rt.ROPE_YARN, factor=16.0, beta_fast=32.0, beta_slow=1.0, orig_ctx=32768,
              attn_factor=0.75)]


def run_append(b, heads, in_t, out_t, rope, positions=None, seed=4, in_place=False):
    g = torch.Generator().manual_seed(seed)
    params = rt.CuqRopeParams(**{"theta": 1e4, **rope})
    plan = rt.RopePlan(params)
    rows = heads + 2 * b.kv_heads
    row = rows * b.hd + 8
    base = torch.randn(max(1, b.n_tok), row, generator=g).to(pu.DT[in_t])
    x = base[: b.n_tok, : rows * b.hd].reshape(b.n_tok, rows, b.hd)
    d = base.cuda()
    size = d.element_size()
    out = torch.full((max(1, b.n_tok), heads * b.hd + 16), 7.0, dtype=pu.DT[out_t], device="cuda")
    pos = None if positions is None else torch.tensor(positions, dtype=torch.int32).cuda()
    k = d.data_ptr() + heads * b.hd * size
    rt.check(lib().cuq_rope_append(plan.handle, b.kvp, b.bp, None if pos is None else ptr(pos),
                                   ptr(d) if in_place else ptr(out), row if in_place else out.shape[1], pu.GGML[out_t],
                                   ptr(d), row, ctypes.c_void_p(k), ctypes.c_void_p(k + b.kv_heads * b.hd * size), row,
                                   pu.GGML[in_t], heads, None))
    torch.cuda.synchronize()
    slots = [n - a + i for a, n in b.seqs for i in range(a)] + [0] * (b.n_tok - b.used)
    p = torch.tensor(slots if positions is None else positions)
    want, w = pu.rotate(x[:, : heads + b.kv_heads], p, params)
    wk, wv = b.k_host.clone(), b.v_host.clone()
    far = torch.zeros_like(b.k_host, dtype=torch.float64)
    for i, (a, n) in enumerate(b.seqs):
        t = b.starts[i]
        sl = slots[t:t + a]
        b.put(wk, i, sl, want[t:t + a, heads:])
        b.put(wv, i, sl, x[t:t + a, heads + b.kv_heads:])
        b.put(far, i, sl, w[t:t + a, heads:])
    got = (d if in_place else out)[: b.n_tok, : heads * b.hd].reshape(b.n_tok, heads, b.hd).double().cpu()
    uo, uc, used = pu.unit(out_t), pu.unit(b.cache), b.used
    sub = 2.0 ** -25 if out_t == "f16" else 0.0
    tol = 2.0 ** -21 * w[:used, :heads] + 1.01 * uo * want[:used, :heads].abs() + sub
    assert ((got[:used] - want[:used, :heads]).abs() <= tol).all()
    if not in_place:
        assert (out[: b.n_tok, heads * b.hd:] == 7).all() and (got[used:] == 7).all()
    else:
        assert torch.equal(got[used:], x[used:, :heads].double())
    gk = b.k.cpu().double()
    # against the exact value: half a step of the cache type and of the rounded 64-bit value it is compared with
    assert ((gk - wk.double()).abs() <= 2.0 ** -21 * far + 2.02 * uc * wk.double().abs() * (far != 0) + 2.0 ** -24 *
            (far != 0)).all()
    assert torch.equal(b.v.cpu(), wv)
    return p


@pytest.mark.parametrize("rope", ROPES)
@pytest.mark.parametrize("types", [("f32", "f32", "f16"), ("f32", "f16", "f16"), ("f16", "f16", "f16"),
                                   ("bf16", "bf16", "bf16"), ("f32", "bf16", "bf16"), ("bf16", "f16", "f16")])
def test_append(rope, types):
    b = pu.Batch([(1, 1), (5, 40), (0, 3), (17, 17), (4, 2), (1, 33)], 2, 64, types[2], 16, tail=3, page_pad=16,
                 holes=[(1, 2)])
    run_append(b, 6, types[0], types[1], rope)


@pytest.mark.parametrize("adjacent", [0, 1])
def test_append_far_positions(adjacent):
    b = pu.Batch([(9, 30)], 1, 128, "f16", 32)
    run_append(b, 3, "f32", "f32", dict(rot_dim=128, adjacent=adjacent),
               positions=[0, 1, 131072, 1000003, (1 << 31) - 1, -5, -(1 << 31), 77, 65536])


@pytest.mark.parametrize("pair", PAIRS)
def test_append_prompt_and_in_place(pair):
    b = pu.Batch([(1100, 1300), (60, 61)], 2, 128, pair[1], 64, tail=1)
    run_append(b, 4, pair[0], pair[0], dict(rot_dim=128))
    b = pu.Batch([(30, 41)], 2, 128, pair[1], 64, tail=1)
    run_append(b, 4, pair[0], pair[0], dict(rot_dim=96, adjacent=1), in_place=True)


def test_append_many_sequences():
    b = pu.Batch([(i % 3, 5 + i % 40) for i in range(700)], 1, 64, "bf16", 16)
    run_append(b, 2, "bf16", "bf16", dict(rot_dim=64))


# ------------------------------------------------------------------ gathered weight ----


def run_mass(seqs, heads, kv_heads, hd, pair, page=16, causal=True, window=0, holes=(), tail=0, last_q=0, decay=1.0,
             seed=0, pad=5):
    t, cache = pair
    b = pu.Batch(seqs, kv_heads, hd, cache, page, seed, tail, holes)
    q, row, qh = queries(b, heads, t, seed + 1)
    scale = hd ** -0.5
    lse = b.attention(qh, scale, causal, window)[1].float()
    g = torch.Generator().manual_seed(seed + 2)
    m0 = torch.rand(len(seqs), kv_heads, b.max_kv + pad, generator=g)
    if decay == 0:
        m0[..., ::3] = math.nan
    m = m0.cuda()
    ld = lse.cuda()
    rt.check(lib().cuq_attention_mass(b.kvp, b.bp, ptr(m), b.max_kv + pad, ptr(q), row, pu.GGML[t], ptr(ld), heads, scale,
                                      int(causal), window, last_q, decay, None))
    rt.check(lib().cuq_paged_status(None))
    got = m.double().cpu()
    add, err = b.mass(qh, lse, scale, causal, window, last_q)
    for i, (_, n) in enumerate(seqs):
        old = m0[i, :, :n].double() * decay if decay else 0.0
        want = old + add[i, :, :n]
        # score sums 2^-17 of sum |q k|, the difference to lse and the exponent 2^-21, and the sum of up to a * group
        # terms in fp32 (pairwise over lanes and tiles: at most 64 roundings in a row)
        tol = 2.0 ** -17 * err[i, :, :n] + 2.0 ** -18 * (add[i, :, :n] + abs(old)) + 1e-30
        assert ((got[i, :, :n] - want).abs() <= tol).all()
        rest = got[i, :, n:]
        old = m0[i, :, n:].double()
        assert torch.equal(rest.nan_to_num(9.0), old.nan_to_num(9.0))


MASS_SEQS = [(1, 1), (1, 700), (2, 17), (5, 64), (32, 1000), (33, 129), (130, 300), (0, 20), (0, 0), (9, 4)]


@pytest.mark.parametrize("geo", GEOS)
@pytest.mark.parametrize("pair", PAIRS)
def test_mass(geo, pair):
    run_mass(MASS_SEQS, *geo, pair, tail=2)


@pytest.mark.parametrize("pair", PAIRS)
@pytest.mark.parametrize("last_q", [1, 8, 32, 100])
def test_mass_of_the_last_queries(last_q, pair):
    run_mass([(32, 500), (100, 1100), (3, 90), (300, 300)], 12, 2, 128, pair, page=64, last_q=last_q, decay=0.0)


@pytest.mark.parametrize("pair", PAIRS)
def test_mass_masks(pair):
    holes = [(0, 0), (1, 3), (2, 0), (2, 5), (0, 28)]
    run_mass([(1, 900), (40, 500), (150, 400)], 12, 2, 128, pair, page=32, window=100, holes=holes, decay=0.5)
    run_mass([(1, 900), (40, 500), (150, 400)], 9, 3, 64, pair, page=32, causal=False, holes=holes, decay=-0.5)
    run_mass([(700, 900)], 4, 2, 64, pair, page=16, decay=0.9)


@pytest.mark.parametrize("pair", PAIRS)
def test_mass_of_many_sequences(pair):
    run_mass([((i % 4), (i * 17) % 70) for i in range(1500)], 4, 2, 64, pair)
    run_mass([(40, 90), (3, 300)], 160, 1, 64, pair, page=32)


def test_mass_repeats_bit_for_bit():
    b = pu.Batch([(300, 900), (20, 2000)], 2, 128, "f16", 64)
    q, row, qh = queries(b, 8, "f16")
    lse = b.attention(qh, 0.1)[1].float().cuda()
    got = []
    for _ in range(3):
        m = torch.zeros(2, 2, b.max_kv, device="cuda")
        rt.check(lib().cuq_attention_mass(b.kvp, b.bp, ptr(m), b.max_kv, ptr(q), row, 1, ptr(lse), 8, 0.1, 1, 0, 0, 1.0,
                                          None))
        got.append(m)
    assert torch.equal(got[0], got[1]) and torch.equal(got[0], got[2])


# ------------------------------------------------------------------ eviction ----


def run_evict(seqs, kv_heads, hd, cache, page, keep, sink, recent, mass=None, holes=(), place="out", seed=0):
    b = pu.Batch([(0, n) for n in seqs], kv_heads, hd, cache, page, seed, holes=holes, page_pad=8)
    g = torch.Generator().manual_seed(seed + 3)
    if mass is None:
        mass = torch.exp(2 * torch.randn(len(seqs), kv_heads, b.max_kv, generator=g))
        mass = mass * (torch.rand(mass.shape, generator=g) > 0.2)
    m = mass.cuda()
    kept = torch.full((len(seqs), kv_heads, keep), 99, dtype=torch.int32, device="cuda")
    new = torch.full((len(seqs),), 99, dtype=torch.int32, device="cuda")
    out = m if place == "in" else torch.full_like(m, 5.0)
    rt.check(lib().cuq_kv_evict(b.kvp, b.bp, ptr(m), b.max_kv, keep, sink, recent, ptr(kept), ptr(new),
                                None if place == "none" else ptr(out), b.max_kv, None))
    torch.cuda.synchronize()
    wk, wv = b.k_host.clone(), b.v_host.clone()
    for i, n in enumerate(seqs):
        rows_k, there = b.rows(b.k_host, i, n)
        rows_v, _ = b.rows(b.v_host, i, n)
        for h in range(kv_heads):
            ids = pu.evict(mass[i, h], n, keep, sink, recent)
            assert kept[i, h].tolist() == ids + [-1] * (keep - len(ids))
            for j, s in enumerate(ids):
                page_id = int(b.table[i, j // page])
                if j != s and there[s] and 0 <= page_id < b.n_pages:
                    at = (h * page + j % page) * hd
                    wk[page_id, at:at + hd] = rows_k[s, h].to(wk.dtype)
                    wv[page_id, at:at + hd] = rows_v[s, h].to(wv.dtype)
            if place != "none":
                o = out[i, h].cpu()
                assert torch.equal(o[: len(ids)].nan_to_num(-1.0), mass[i, h][ids].nan_to_num(-1.0))
                assert (o[len(ids):n] == 0).all()
                rest = mass[i, h, n:] if place == "in" else torch.full((b.max_kv - n,), 5.0)
                assert torch.equal(o[n:], rest)
    assert new.tolist() == [min(n, keep) for n in seqs]
    assert torch.equal(b.k.cpu(), wk) and torch.equal(b.v.cpu(), wv)


@pytest.mark.parametrize("cache,hd", [("f16", 64), ("bf16", 128)])
@pytest.mark.parametrize("place", ["out", "in", "none"])
def test_evict(cache, hd, place):
    run_evict([100, 33, 32, 31, 0, 1, 1500, 4099], 3, hd, cache, 16, 32, 4, 8, place=place)
    run_evict([5000, 700], 2, hd, cache, 64, 601, 0, 0, place=place, seed=1)


@pytest.mark.parametrize("keep,sink,recent", [(1, 0, 0), (1, 1, 0), (1, 0, 1), (64, 32, 32), (999, 3, 900), (1000, 0, 0),
                                              (2000, 10, 10)])
def test_evict_budgets(keep, sink, recent):
    run_evict([1000, 999, 65], 2, 64, "f16", 32, keep, sink, recent)


@pytest.mark.parametrize("cache,hd", [("f16", 64), ("bf16", 128)])
def test_evict_long(cache, hd):
    run_evict([70001, 40000], 1, hd, cache, 256, 30011, 4, 100)


def test_evict_ties_and_odd_masses():
    n = 600
    m = torch.zeros(1, 4, n)
    m[0, 1] = torch.arange(n).remainder(3).float()
    m[0, 2, ::2], m[0, 2, 1::2] = -0.0, 0.0
    m[0, 3] = torch.randn(n, generator=torch.Generator().manual_seed(1))
    m[0, 3, 5::7], m[0, 3, 6::11], m[0, 3, 8::13] = math.nan, math.inf, -math.inf
    for keep in (1, 50, 300, 595):
        run_evict([n], 4, 64, "f16", 16, keep, 0, 0, mass=m.clone())
        run_evict([n], 4, 64, "f16", 16, keep, 1, 0, mass=m.clone(), place="in")


@pytest.mark.parametrize("n", [700, 9000])
@pytest.mark.parametrize("place", ["in", "out"])
def test_evict_edges_between_bits(place, n):
    """Groups of equal masses that differ from bit 27, 20, 9 or 0 on, kept to a group's last member, one short of it
    and one past it."""
    m = torch.zeros(1, 4, n, dtype=torch.int32)
    group = torch.randint(0, 5, (4, n), generator=torch.Generator().manual_seed(7))
    for h, bit in enumerate((27, 20, 9, 0)):
        m[0, h] = 0x20000000 + (group[h] << bit).int()
    m = m.view(torch.float32)
    m[0, 3, ::2] *= -1
    for top in (1, 2, 4):
        edge = int((group[0] >= top).sum())
        for keep in (edge - 1, edge, edge + 1):
            run_evict([n], 4, 64, "bf16", 32, keep, 0, 0, mass=m.clone(), place=place)
    for h in range(4):  # the boundary right behind each head's own groups
        run_evict([n], 4, 64, "bf16", 32, int((group[h] >= 3).sum()), 0, 0, mass=m.clone(), place=place)


def test_evict_holes_stay_out_of_it():
    run_evict([300, 200], 2, 64, "f16", 16, 100, 4, 16, holes=[(0, 3), (0, 9), (1, 0)])


# ------------------------------------------------------------------ together ----


@pytest.mark.parametrize("pair", PAIRS)
def test_a_served_batch_from_prompt_to_eviction(pair):
    """Prompts appended and attended, the gathered weight, an eviction per head, then decode steps over what is left."""
    L = lib()
    t, cache = pair
    heads, kvh, hd, page, keep = 4, 2, 64, 16, 48
    rope = rt.CuqRopeParams(rot_dim=32, theta=1e4)
    plan = rt.RopePlan(rope)
    lens = [90, 37, 130]
    b = pu.Batch([(n, n) for n in lens], kvh, hd, cache, page, capacity=8)
    g = torch.Generator().manual_seed(2)
    mass = torch.zeros(3, kvh, b.max_kv, device="cuda")
    model = [[None] * kvh for _ in lens]  # per sequence and head: 64-bit (k, v) rows
    scale, row = hd ** -0.5, (heads + 2 * kvh) * hd

    def step(seqs, pos):
        b.seqs = seqs
        b.starts = [0]
        for a, _ in seqs:
            b.starts.append(b.starts[-1] + a)
        n = b.n_tok = b.used = b.starts[-1]
        b.d_start.copy_(torch.tensor(b.starts, dtype=torch.int32))
        b.desc.n_tok, b.desc.max_q = n, max(a for a, _ in seqs)
        x = torch.randn(n, heads + 2 * kvh, hd, generator=g).to(pu.DT[t])
        d, p = x.cuda(), torch.tensor(pos, dtype=torch.int32).cuda()
        q = torch.empty(n, heads * hd, dtype=pu.DT[t], device="cuda")
        size = d.element_size()
        k = d.data_ptr() + heads * hd * size
        rt.check(L.cuq_rope_append(plan.handle, b.kvp, b.bp, ptr(p), ptr(q), heads * hd, pu.GGML[t], ptr(d), row,
                                   ctypes.c_void_p(k), ctypes.c_void_p(k + kvh * hd * size), row, pu.GGML[t], heads,
                                   None))
        out, lse = attend(b, heads, t, q, heads * hd, scale)
        rt.check(L.cuq_attention_mass(b.kvp, b.bp, ptr(mass), b.max_kv, ptr(q), heads * hd, pu.GGML[t], ptr(lse), heads,
                                      scale, 1, 0, 0, 1.0, None))
        torch.cuda.synchronize()
        # the model rotates in 64 bits and rounds as the cache does
        y, _ = pu.rotate(x[:, : heads + kvh], torch.tensor(pos), rope)
        qr = y[:, :heads].to(pu.DT[t]).double()
        kr, vr = y[:, heads:].to(pu.DT[cache]).double(), x[:, heads + kvh:].to(pu.DT[cache]).double()
        got = out[:n].view(n, heads, hd).double().cpu()
        for i, (a, _) in enumerate(seqs):
            s = b.starts[i]
            for h in range(kvh):
                old = model[i][h]
                new = (kr[s:s + a, h], vr[s:s + a, h])
                model[i][h] = new if old is None else tuple(torch.cat(z) for z in zip(old, new))
                kk, vv = model[i][h]
                m = kk.shape[0]
                ok = torch.arange(m)[None] <= torch.arange(m - a, m)[:, None]
                for gq in range(heads // kvh):
                    w = torch.softmax((qr[s:s + a, h * 2 + gq] @ kk.T * scale).masked_fill(~ok, -math.inf), 1)
                    want = w @ vv
                    u = pu.unit(t)
                    # a key or query may round the other way (a whole step of its type, on every term)
                    uc = pu.unit(cache)
                    tol = 24 * uc * (w @ vv.abs()) + 2 * u * want.abs() + 1e-6
                    assert ((got[s:s + a, h * 2 + gq] - want).abs() <= tol).all()

    def set_len(n):
        b.d_len.copy_(torch.tensor(n, dtype=torch.int32))

    set_len(lens)
    step([(n, n) for n in lens], [p for n in lens for p in range(n)])
    assert abs(float(mass.sum()) - heads * sum(lens)) < 1e-2 * heads * sum(lens)  # every query's weights sum to one
    kept = torch.empty(3, kvh, keep, dtype=torch.int32, device="cuda")
    new = torch.empty(3, dtype=torch.int32, device="cuda")
    before = mass.cpu()
    rt.check(L.cuq_kv_evict(b.kvp, b.bp, ptr(mass), b.max_kv, keep, 4, 8, ptr(kept), ptr(new), ptr(mass), b.max_kv, None))
    torch.cuda.synchronize()
    now = [min(n, keep) for n in lens]
    assert new.tolist() == now
    for i, n in enumerate(lens):
        for h in range(kvh):
            ids = pu.evict(before[i, h], n, keep, 4, 8)
            assert kept[i, h, : now[i]].tolist() == ids
            model[i][h] = tuple(z[ids] for z in model[i][h])
    for j in range(5):  # single tokens, at their own rotary positions, behind the kept slots
        set_len([n + j + 1 for n in now])
        step([(1, n + j + 1) for n in now], [n + j for n in lens])


def test_graph_replay_follows_the_arrays():
    """One captured graph of append and attention, replayed while lengths and tables change on the device."""
    L = lib()
    b = pu.Batch([(1, 40), (1, 300), (1, 7)], 2, 128, "bf16", 16, capacity=64)
    heads, hd = 8, 128
    row = (heads + 4) * hd
    plan = rt.RopePlan(rt.CuqRopeParams(rot_dim=128, theta=1e4))
    d = torch.randn(3, row, device="cuda").bfloat16()
    q = torch.empty(3, heads * hd, dtype=torch.bfloat16, device="cuda")
    out, lse = torch.empty_like(q), torch.empty(3, heads, device="cuda")
    b.desc.max_kv = b.max_kv
    need = L.cuq_attention_paged_workspace(b.kvp, b.bp, heads, 30)
    ws = torch.empty(max(1, need), dtype=torch.uint8, device="cuda")
    mass = torch.zeros(3, 2, b.max_kv, device="cuda")

    def calls(s):
        rt.check(L.cuq_rope_append(plan.handle, b.kvp, b.bp, None, ptr(q), heads * hd, 30, ptr(d), row,
                                   ctypes.c_void_p(d.data_ptr() + heads * hd * 2),
                                   ctypes.c_void_p(d.data_ptr() + (heads + 2) * hd * 2), row, 30, heads, s))
        rt.check(L.cuq_attention_paged(b.kvp, b.bp, ptr(out), heads * hd, ptr(q), heads * hd, 30, ptr(lse), heads, 0.1, 1, 0,
                                       ptr(ws), need, s))
        rt.check(L.cuq_attention_mass(b.kvp, b.bp, ptr(mass), b.max_kv, ptr(q), heads * hd, 30, ptr(lse), heads, 0.1, 1, 0,
                                      0, 0.0, s))

    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        calls(stream.cuda_stream)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        calls(torch.cuda.current_stream().cuda_stream)
    for lens in ([41, 301, 8], [42, 302, 9], [1, 350, 64], [0, 17, 0]):
        b.d_len.copy_(torch.tensor(lens, dtype=torch.int32))
        d.normal_()
        graph.replay()
        torch.cuda.synchronize()
        b.seqs = [(1, n) for n in lens]
        b.k_host, b.v_host = b.k.cpu(), b.v.cpu()
        check_attention(b, heads, "bf16", out, lse, q.view(3, heads, hd).cpu(), 0.1)
        for i, n in enumerate(lens):  # each head's weights sum to one over the live slots
            assert abs(float(mass[i, :, :n].sum()) - (heads if n else 0)) < 2.0 ** -10 * heads


@pytest.mark.parametrize("slots", [512, 16384])
@pytest.mark.parametrize("pair", PAIRS)
def test_graph_replay_of_single_tokens(pair, slots):
    """A captured decode step under a bound of few and of many slots (one launch, or runs and the merge), lengths changing."""
    t, cache = pair
    L, heads, hd = lib(), 9, 64
    b = pu.Batch([(1, 40), (1, 500), (1, 7), (1, 129)], 3, hd, cache, 16, seed=41, tail=1)
    wide = torch.full((4, slots // 16), -1, dtype=torch.int32)
    wide[:, : b.table.shape[1]] = b.table
    d_wide = wide.cuda()
    b.desc.pages, b.desc.pages_stride, b.desc.max_kv = d_wide.data_ptr(), slots // 16, slots
    need = L.cuq_attention_paged_workspace(b.kvp, b.bp, heads, pu.GGML[t])
    assert (need == 0) == (slots == 512)
    ws = torch.full((max(1, need),), 255, dtype=torch.uint8, device="cuda")
    q, row, qh = queries(b, heads, t, 42)
    out = torch.full((b.n_tok, heads * hd), 7.0, dtype=pu.DT[t], device="cuda")
    lse = torch.full((b.n_tok, heads), 7.0, device="cuda")

    def call(s):
        rt.check(L.cuq_attention_paged(b.kvp, b.bp, ptr(out), heads * hd, ptr(q), row, pu.GGML[t], ptr(lse), heads, 0.125, 1,
                                       0, ptr(ws) if need else None, need, s))

    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    call(stream.cuda_stream)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        for _ in range(3):
            call(torch.cuda.current_stream().cuda_stream)
    for lens in ([40, 500, 7, 129], [1, 2, 0, 16], [33, 17, 7, 1], [0, 0, 0, 0]):
        b.d_len.copy_(torch.tensor(lens, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        b.seqs = [(1, n) for n in lens]
        check_attention(b, heads, t, out, lse, qh, 0.125)


def test_two_calls_at_once():
    """Two batches on two streams with a workspace each."""
    bs = [pu.Batch([(1, 3000 + 500 * i), (200, 700)], 2, 128, "f16", 64, seed=i) for i in range(2)]
    qs = [queries(b, 8, "f16", seed=20 + i) for i, b in enumerate(bs)]
    streams = [torch.cuda.Stream() for _ in bs]
    L = lib()
    outs, spaces = [], []
    for b in bs:
        need = L.cuq_attention_paged_workspace(b.kvp, b.bp, 8, 1)
        spaces.append((torch.empty(max(1, need), dtype=torch.uint8, device="cuda"), need))
        outs.append((torch.full((b.n_tok, 8 * 128), 7.0, dtype=torch.float16, device="cuda"),
                     torch.full((b.n_tok, 8), 7.0, device="cuda")))
    torch.cuda.synchronize()
    for _ in range(5):
        for b, (q, row, _), s, (o, l), (w, need) in zip(bs, qs, streams, outs, spaces):
            rt.check(L.cuq_attention_paged(b.kvp, b.bp, ptr(o), 1024, ptr(q), row, 1, ptr(l), 8, 0.1, 1, 0, ptr(w), need,
                                           s.cuda_stream))
    torch.cuda.synchronize()
    for b, (_, _, qh), (o, l) in zip(bs, qs, outs):
        check_attention(b, 8, "f16", o, l, qh, 0.1)
