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
from .test_gpu_paged import PAIRS, check_attention, run_attention

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
