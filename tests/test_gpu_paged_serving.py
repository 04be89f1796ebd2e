"""The paged-cache ops as a server runs them: captured steps whose batch changes, many items a CTA, and what a wait that
gives up leaves behind.  Tolerances are those of test_gpu_paged.py unless a test derives its own."""
import ctypes
import math
from decimal import Decimal, getcontext

import pytest
import torch

from anedvd_b200 import runtime as rt

from . import paged_util as pu
from .gpu_util import lib, ptr
from .test_gpu_paged import PAIRS, attend, check_attention, run_attention

pytestmark = pytest.mark.gpu


class Step:
    """Append, attention and gathered weight of one batch, with the buffers that a server keeps for them."""

    def __init__(self, b, heads, pair, window=0):
        t, _ = pair
        self.b, self.heads, self.t, self.window = b, heads, t, window
        self.plan = rt.RopePlan(rt.CuqRopeParams(rot_dim=b.hd, theta=1e4))
        dt, self.cols = pu.DT[t], heads * b.hd
        self.x = torch.zeros(b.n_tok, (heads + 2 * b.kv_heads) * b.hd, dtype=dt, device="cuda")
        self.q, self.out = (torch.full((b.n_tok, self.cols), 7.0, dtype=dt, device="cuda") for _ in range(2))
        self.lse = torch.full((b.n_tok, heads), 7.0, device="cuda")
        self.mass = torch.zeros(len(b.seqs), b.kv_heads, b.max_kv, device="cuda")
        self.need = lib().cuq_attention_paged_workspace(b.kvp, b.bp, heads, pu.GGML[t])
        self.space = torch.full((max(1, self.need),), 255, dtype=torch.uint8, device="cuda")

    def calls(self, stream):
        b, L, ty, row = self.b, rt.load(), pu.GGML[self.t], self.x.shape[1]
        k = self.x.data_ptr() + self.cols * self.x.element_size()
        v = k + b.kv_heads * b.hd * self.x.element_size()
        rt.check(L.cuq_rope_append(self.plan.handle, b.kvp, b.bp, None, ptr(self.q), self.cols, ty, ptr(self.x), row,
                                   ctypes.c_void_p(k), ctypes.c_void_p(v), row, ty, self.heads, stream))
        rt.check(L.cuq_attention_paged(b.kvp, b.bp, ptr(self.out), self.cols, ptr(self.q), self.cols, ty, ptr(self.lse),
                                       self.heads, 0.1, 1, self.window, ptr(self.space), self.need, stream))
        rt.check(L.cuq_attention_mass(b.kvp, b.bp, ptr(self.mass), b.max_kv, ptr(self.q), self.cols, ty, ptr(self.lse),
                                      self.heads, 0.1, 1, self.window, 0, 0.0, stream))

    def check(self):
        b = self.b
        b.k_host, b.v_host = b.k.cpu(), b.v.cpu()
        q = self.q[: b.n_tok].view(b.n_tok, self.heads, b.hd).cpu()
        # only rows of the batch are the model's: the others keep what an earlier step left there
        out, lse = self.out.clone(), self.lse.clone()
        out[b.used:], lse[b.used:] = 7.0, 7.0
        check_attention(b, self.heads, self.t, out, lse, q, 0.1, window=self.window)
        for i, (a, n) in enumerate(b.seqs):  # each row's weights sum to one over the live slots
            want = self.heads * min(a, n)
            assert abs(float(self.mass[i, :, :n].double().sum()) - want) <= 2.0 ** -10 * max(1, want)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("pair", PAIRS)
def test_captured_mixed_steps_follow_the_batch(pair, hd):
    """Chunks beside single tokens in one captured graph (both attention kernels and the merge): which sequence has the
    chunk, the lengths, the queries and the cached rows all change between replays, three steps behind one another."""
    b = pu.Batch([(48, 200), (48, 300), (48, 48), (48, 90)], 2, hd, pair[1], 16, seed=3, tail=0)
    b.n_tok = b.desc.n_tok = 64
    step = Step(b, 8, pair)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    step.calls(stream.cuda_stream)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        for _ in range(3):  # the later steps write the same rows again
            step.calls(torch.cuda.current_stream().cuda_stream)
    g = torch.Generator(device="cuda").manual_seed(5)
    for seqs in ([(40, 150), (1, 300), (1, 20), (1, 90)], [(1, 151), (48, 300), (1, 21), (2, 90)],
                 [(2, 150), (0, 300), (48, 48), (1, 1)], [(1, 200), (1, 299), (1, 48), (1, 89)],
                 [(10, 150), (10, 30), (30, 48), (3, 2)], [(0, 200), (1, 7), (0, 0), (0, 1)]):
        b.seqs, b.starts = seqs, [0]
        for a, _ in seqs:
            b.starts.append(b.starts[-1] + a)
        b.used = b.starts[-1]
        b.d_start.copy_(torch.tensor(b.starts, dtype=torch.int32))
        b.d_len.copy_(torch.tensor([n for _, n in seqs], dtype=torch.int32))
        step.x.normal_(generator=g)
        graph.replay()
        torch.cuda.synchronize()
        step.check()


def test_every_stream_is_told_of_a_wait_that_gave_up():
    """A wait that nothing ends gives up after its limit; each polled stream is told once, whoever asks first, and the
    next calls are as before."""
    L = lib()
    one, two = torch.cuda.Stream().cuda_stream, torch.cuda.Stream().cuda_stream
    for s in (one, two, None):
        L.cuq_paged_status(s)  # whatever came before
        assert L.cuq_paged_status(s) == rt.OK
    rt.check(L.cuq_paged_wait_probe(1000, one))
    assert L.cuq_paged_status(one) == rt.ETIMEOUT
    assert "gave up" in rt.last_error()
    assert L.cuq_paged_status(one) == rt.OK
    assert L.cuq_paged_status(two) == rt.ETIMEOUT
    rt.check(L.cuq_paged_wait_probe(500, two))
    rt.check(L.cuq_paged_wait_probe(500, two))
    assert L.cuq_paged_status(two) == rt.ETIMEOUT
    for s in (one, None):
        assert L.cuq_paged_status(s) == rt.ETIMEOUT
        assert L.cuq_paged_status(s) == rt.OK
    assert L.cuq_paged_status(two) == rt.OK
    run_attention([(1, 70), (40, 90)], 4, 2, 64, ("f16", "f16"))


def test_a_give_up_in_a_graph_is_told_where_it_is_replayed():
    L = lib()
    stream, other = torch.cuda.Stream(), torch.cuda.Stream()
    for s in (stream.cuda_stream, other.cuda_stream, None):
        L.cuq_paged_status(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        rt.check(L.cuq_paged_wait_probe(500, torch.cuda.current_stream().cuda_stream))
    assert L.cuq_paged_status(other.cuda_stream) == rt.OK
    for _ in range(2):
        with torch.cuda.stream(other):
            graph.replay()
        assert L.cuq_paged_status(other.cuda_stream) == rt.ETIMEOUT
        assert L.cuq_paged_status(other.cuda_stream) == rt.OK
    assert L.cuq_paged_status(None) == rt.ETIMEOUT


def turns(params):
    """Turns per position of each pair, to 50 digits."""
    getcontext().prec = 50
    two_pi = 2 * Decimal("3.14159265358979323846264338327950288419716939937510582097494459")
    rot, theta = params.rot_dim, Decimal(float(params.theta))
    f = [(-(2 * Decimal(j) / rot) * theta.ln()).exp() for j in range(rot // 2)]
    if params.scaling == rt.ROPE_LINEAR:
        f = [x / Decimal(float(params.factor)) for x in f]
    return [x / two_pi for x in f]


@pytest.mark.parametrize("theta", [1e4, 1e6])
@pytest.mark.parametrize("scaling", [rt.ROPE_NONE, rt.ROPE_LINEAR])
def test_angles_hold_at_the_farthest_positions(scaling, theta):
    """cos and sin themselves (pairs (1, 0)) at positions up to 2^31.  The angle is off by 2^-32 turns from the table and
    pi 2^-25 from its rounding to fp32, the functions by 2 steps of a value below one, 2^-23 in all."""
    hd, n = 128, 96
    params = rt.CuqRopeParams(rot_dim=hd, theta=theta, scaling=scaling, factor=3.0)
    plan = rt.RopePlan(params)
    b = pu.Batch([(n, n)], 1, hd, "f16", 16)
    pos = [(-1) ** i * ((1 << 31) - 1 - 12345677 * i) for i in range(n)]
    x = torch.zeros(n, 3, hd, device="cuda")
    x[:, 0, : hd // 2] = 1.0
    q = torch.empty(n, hd, device="cuda")
    at = torch.tensor(pos, dtype=torch.int32, device="cuda")
    rt.check(lib().cuq_rope_append(plan.handle, b.kvp, b.bp, ptr(at), ptr(q), hd, 0, ptr(x), 3 * hd,
                                   ctypes.c_void_p(x.data_ptr() + 4 * hd), ctypes.c_void_p(x.data_ptr() + 8 * hd), 3 * hd,
                                   0, 1, None))
    got = q.double().cpu()
    tol = 2 * math.pi * 2.0 ** -32 + math.pi * 2.0 ** -25 + 2.0 ** -23
    for j, t in enumerate(turns(params)):
        angle = [2 * math.pi * float(p * t % 1) for p in pos]
        for k, f in ((j, math.cos), (j + hd // 2, math.sin)):
            want = torch.tensor([f(a) for a in angle], dtype=torch.float64)
            assert float((got[:, k] - want).abs().max()) <= tol, (j, k)


def wide_table(b, slots):
    """The same caches under a bound of `slots` slots, which asks for runs and the merge."""
    wide = torch.full((len(b.seqs), slots // b.page), -1, dtype=torch.int32)
    wide[:, : b.table.shape[1]] = b.table
    b.d_wide = wide.cuda()
    b.desc.pages, b.desc.pages_stride, b.desc.max_kv = b.d_wide.data_ptr(), slots // b.page, slots


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("seqs,form", [
    ([(1, 300), (1, 900), (1, 77)], "cluster"), ([(1, 300), (1, 900), (3, 2000)], "runs"), ([(100, 500)], "whole"),
    ([(40, 1500)], "split"), ([(1, 700), (100, 500), (2, 300)], "mixed")])
def test_fp32_queries_keep_what_fp32_holds(seqs, form, hd):
    """Against 64 bits, relative to sum p |v| / sum p = mag, each row at its own length.  Values are 1 + noise, so that what
    an accumulator cuts off adds up.  Counted, with T = scale sum |q k| (below 2.5 here) and a cut of at most 2^-22 of the
    sum at each of the matrix instructions behind one another (two a step, one of them in the other half's place):
      scores: hd / 16 steps and two roundings more, (hd / 16 + 2) 2^-22 T, twice (numerator and sum);
      probabilities: the exponent's rounding below 16, 2^-21, the exponential 2^-22 and the split 2^-22: below 2^-20;
      products with V: 16 instructions a tile of 128 slots, up to 40 in a warp's run: 40 * 2^-22;
      sums of up to 64 probabilities a thread, and the parts' weights: 2^-18.
    The mean square counts cuts as half a step on average, growing with the sum (a quarter of the bound: 10 * 2^-22 = 2.4e-6
    at most, 16 instructions 1e-6), and the rest as independent over the slots.  Probabilities rounded to fp16
    without their low parts, worked out for these inputs, give 1.3e-5 at 300 slots and 8.5e-6 at 900 (root mean square)."""
    b = pu.Batch(seqs, 2, hd, "f16", 16, seed=31)
    for host, dev in ((b.k_host, b.k), (b.v_host, b.v)):
        if host is b.v_host:
            host.mul_(0.5).add_(1.0)
        dev.copy_(host)
    if form == "runs":
        wide_table(b, 16384)
    heads, scale = 8, 1.0 / 64
    g = torch.Generator().manual_seed(32)
    q = torch.randn(b.n_tok, heads, hd, generator=g)
    need = lib().cuq_attention_paged_workspace(b.kvp, b.bp, heads, 0)
    assert (need == 0) == (form in ("cluster", "whole"))
    out, lse = attend(b, heads, "f32", q.cuda().view(b.n_tok, -1), heads * hd, scale)
    want, wl, mag, top = b.attention(q, scale)
    assert float(top.max()) < 2.5
    off = (out.view(b.n_tok, heads, hd).double().cpu() - want).abs() / mag
    tol = 2 * top[..., None] * (hd / 16 + 2) * 2.0 ** -22 + 2.0 ** -20 + 40 * 2.0 ** -22 + 2.0 ** -18
    assert float((off - tol).max()) <= 0, float((off / tol).max())
    for i, (a, n) in enumerate(seqs):
        t = b.starts[i]
        if 300 <= n <= 900:
            assert float(off[t:t + a].square().mean().sqrt()) <= 2.4e-6
    assert float((lse.double().cpu() - wl).abs().max()) <= 2.5 * (hd / 16 + 2) * 2.0 ** -22 + 2.0 ** -18 + 2.0 ** -20


@pytest.mark.parametrize("pair", PAIRS)
@pytest.mark.parametrize("long", [False, True])
def test_mass_of_more_items_than_a_block_lists(pair, long):
    """More than 64 items of 256 slots for every block of the GPU: neighbouring ones where the queries are few, dealt out
    where some sequence has more than 128 rows; ragged lengths, empty caches, sequences without tokens.  All caches share
    a few pages, which this operator only reads."""
    t, cache = pair
    heads, kvh, hd, page, n_seqs = 4, 2, 64, 256, 640
    g = torch.Generator().manual_seed(51)
    lens = torch.randint(1500, 3001, (n_seqs,), generator=g).tolist()
    toks = torch.randint(1, 4, (n_seqs,), generator=g).tolist()
    for i in range(0, n_seqs, 37):
        toks[i] = 90 if long else 0
    for i in range(5, n_seqs, 41):
        lens[i] = 0
    for i in range(7, n_seqs, 43):
        toks[i] = 0
    lens = [max(n, a) if n else 0 for n, a in zip(lens, toks)]
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    assert sum(-(-n // 256) for n in lens) * kvh > 64 * sms
    n_pages, cols = 40, 13
    table = torch.randint(0, n_pages, (n_seqs, cols), generator=g).int()
    table[::53, 3] = -1  # holes
    starts = [0]
    for a in toks:
        starts.append(starts[-1] + a)
    n_tok, max_kv, max_q = starts[-1], max(lens), max(toks)
    assert (max_q * 2 > 128) == long
    k = torch.randn(n_pages, kvh, page, hd, generator=g).to(pu.DT[cache]).cuda()
    q = (1.5 * torch.randn(n_tok, heads, hd, generator=g)).to(pu.DT[t]).cuda()
    dev = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in (starts, lens)] + [table.cuda()]
    kv = rt.CuqPagedKv(k=k.data_ptr(), v=k.data_ptr(), type=pu.GGML[cache], n_pages=n_pages, page_size=page, kv_heads=kvh,
                       head_dim=hd, page_stride=0)
    batch = rt.CuqBatch(q_start=dev[0].data_ptr(), kv_len=dev[1].data_ptr(), pages=dev[2].data_ptr(), n_seqs=n_seqs,
                        n_tok=n_tok, pages_stride=cols, max_q=max_q, max_kv=max_kv)
    # the definition in 64 bits; terms and their error weights as in paged_util.Batch.mass
    scale = hd ** -0.5
    lse = torch.zeros(n_tok, heads, dtype=torch.float64, device="cuda")
    parts = []
    for i, (a, n) in enumerate(zip(toks, lens)):
        if not a or not n:
            parts.append(None)
            continue
        slot = torch.arange(n, device="cuda")
        ids = dev[2][i].long()[slot // page]
        rows = k[ids.clamp(min=0), :, slot % page].double()                           # [n][kvh][hd]
        qq = q[starts[i]:starts[i + 1]].double().view(a, kvh, heads // kvh, hd)
        x = torch.einsum("akgd,nkd->kgan", qq, rows) * scale
        ok = (ids >= 0) & (slot <= torch.arange(n - a, n, device="cuda")[:, None])
        x = x.masked_fill(~ok, -math.inf)
        far = torch.einsum("akgd,nkd->kgan", qq.abs(), rows.abs()) * scale
        lse[starts[i]:starts[i + 1]] = torch.logsumexp(x, 3).permute(2, 0, 1).reshape(a, heads)
        parts.append((x, far))
    ls = lse.float()
    mass = torch.rand(n_seqs, kvh, max_kv, generator=g).cuda()
    before = mass.double()
    rt.check(lib().cuq_attention_mass(ctypes.byref(kv), ctypes.byref(batch), ptr(mass), max_kv, ptr(q), heads * hd,
                                      pu.GGML[t], ptr(ls), heads, scale, 1, 0, 0, 0.5, None))
    rt.check(lib().cuq_paged_status(None))
    got = mass.double()
    for i, (a, n) in enumerate(zip(toks, lens)):
        assert torch.equal(got[i, :, n:], before[i, :, n:])
        add = err = torch.zeros(kvh, n, dtype=torch.float64, device="cuda")
        if parts[i]:
            x, far = parts[i]
            ll = ls[starts[i]:starts[i + 1]].double().view(a, kvh, heads // kvh).permute(1, 2, 0)[..., None]
            p = torch.exp(x - ll)
            add, err = p.sum((1, 2)), (p * (far + ll.abs())).sum((1, 2))
        want = 0.5 * before[i, :, :n] + add
        tol = 2.0 ** -17 * err + 2.0 ** -18 * want + 1e-30
        assert ((got[i, :, :n] - want).abs() <= tol).all(), i


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("form", ["cluster", "runs"])
def test_few_rows_round_the_output_alone(form, t, hd):
    """Decode steps in 16 bits: half a step of the output, and beside it what fp32 queries are allowed above, with
    probabilities of two 16-bit operands (u^2 of themselves, 2^-16 in bf16, in the products alone).  One rounded operand is
    off by up to u of each probability, and outputs near zero show it."""
    seqs = [(1, 300), (1, 900), (2, 150)]
    b = pu.Batch(seqs, 2, hd, t, 16, seed=61)
    if form == "runs":
        wide_table(b, 16384)
    heads, scale = 8, 1.0 / 64
    q = torch.randn(b.n_tok, heads, hd, generator=torch.Generator().manual_seed(62)).to(pu.DT[t])
    need = lib().cuq_attention_paged_workspace(b.kvp, b.bp, heads, pu.GGML[t])
    assert (need == 0) == (form == "cluster")
    out, _ = attend(b, heads, t, q.cuda().view(b.n_tok, -1), heads * hd, scale)
    want, _, mag, top = b.attention(q, scale)
    off = (out.view(b.n_tok, heads, hd).double().cpu() - want).abs()
    u = pu.unit(t)
    tol = mag * (2 * top[..., None] * (hd / 16 + 2) * 2.0 ** -22 + 2.0 ** -20 + 40 * 2.0 ** -22 + 2.0 ** -18 + u * u)
    tol = tol + 1.01 * u * want.abs() + 2.0 ** -25
    assert float((off - tol).max()) <= 0, float((off / tol).max())
