"""A paged cache and a batch on the device for the tests, with a 64-bit model of what the paged ops compute."""
import ctypes
import math

import torch

from anedvd_b200 import runtime as rt

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
GGML = {"f32": 0, "f16": 1, "bf16": 30}


def unit(name):
    """Half a step of the type, relative to the value."""
    return torch.finfo(DT[name]).eps / 2


class Batch:
    """`seqs`: [(new tokens, cache length with them)].  Pools are random; pages are handed out in a random order with
    spare ones in between; `holes`: (sequence, table column) entries replaced by ids outside the pool."""

    def __init__(self, seqs, kv_heads, hd, cache="f16", page=16, seed=0, tail=0, holes=(), page_pad=0, capacity=0,
                 device="cuda"):
        g = torch.Generator().manual_seed(seed)
        self.seqs, self.kv_heads, self.hd, self.cache, self.page = list(seqs), kv_heads, hd, cache, page
        self.device = device
        self.max_q = max([a for a, _ in seqs] + [0])
        self.max_kv = max([b for _, b in seqs] + [0]) + capacity
        cols = max(1, -(-self.max_kv // page))
        need = [-(-(b + capacity) // page) for _, b in seqs]
        self.n_pages = sum(need) + 2
        ids = torch.randperm(self.n_pages, generator=g).tolist()
        table = torch.full((len(seqs), cols), 1 << 30, dtype=torch.int32)  # past a sequence's end: no page
        at = 0
        for b, n in enumerate(need):
            table[b, :n] = torch.tensor(ids[at:at + n], dtype=torch.int32)
            at += n
        for i, (b, c) in enumerate(holes):
            table[b, c] = [-1, self.n_pages, -(1 << 31), (1 << 31) - 1][i % 4]
        starts = [0]
        for a, _ in seqs:
            starts.append(starts[-1] + a)
        self.used, self.n_tok = starts[-1], starts[-1] + tail
        self.stride = kv_heads * page * hd + page_pad
        pool = lambda: torch.randn(self.n_pages, self.stride, generator=g).to(DT[cache])  # noqa: E731
        self.k_host, self.v_host = pool(), pool()
        self.table, self.starts = table, starts
        to = lambda x: x.to(device)  # noqa: E731
        self.k, self.v, self.d_table = to(self.k_host.clone()), to(self.v_host.clone()), to(table)
        self.d_start = to(torch.tensor(starts, dtype=torch.int32))
        self.d_len = to(torch.tensor([b for _, b in seqs], dtype=torch.int32))
        self.kv_desc = rt.CuqPagedKv(k=self.k.data_ptr(), v=self.v.data_ptr(), type=GGML[cache], n_pages=self.n_pages,
                                     page_size=page, kv_heads=kv_heads, head_dim=hd, page_stride=self.stride)
        self.desc = rt.CuqBatch(q_start=self.d_start.data_ptr(), kv_len=self.d_len.data_ptr(),
                                pages=self.d_table.data_ptr(), n_seqs=len(seqs), n_tok=self.n_tok, pages_stride=cols,
                                max_q=self.max_q, max_kv=self.max_kv)

    @property
    def kvp(self):
        return ctypes.byref(self.kv_desc)

    @property
    def bp(self):
        return ctypes.byref(self.desc)

    def rows(self, pool, b, n):
        """[n][kv_heads][hd] rows of sequence b's first n slots in a [pages][stride] host pool, and whether each is
        there."""
        slot = torch.arange(n)
        page = self.table[b, slot // self.page].long()
        there = (page >= 0) & (page < self.n_pages)
        p = pool[:, : self.kv_heads * self.page * self.hd].reshape(self.n_pages, self.kv_heads, self.page, self.hd)
        return p[page.clamp(0, self.n_pages - 1), :, slot % self.page].double(), there

    def put(self, pool, b, slot, rows):
        """Write rows [n][kv_heads][hd] at slots of sequence b of a host pool; rows on a hole are dropped."""
        p = pool[:, : self.kv_heads * self.page * self.hd].reshape(self.n_pages, self.kv_heads, self.page, self.hd)
        for i, s in enumerate(slot):
            if s < 0:
                continue
            page = int(self.table[b, s // self.page])
            if 0 <= page < self.n_pages:
                p[page, :, s % self.page] = rows[i].to(pool.dtype)
        if p.data_ptr() != pool.data_ptr():
            pool[:, : self.kv_heads * self.page * self.hd] = p.reshape(self.n_pages, -1)

    def seen(self, b, causal, window):
        """[new tokens][slots]: who sees what."""
        a, n = self.seqs[b]
        pos, key = torch.arange(n - a, n)[:, None], torch.arange(n)[None]
        _, there = self.rows(self.k_host, b, n)
        ok = there[None] & (pos >= 0)
        if causal:
            ok = ok & (key <= pos)
            if window:
                ok = ok & (key > pos - window)
        return ok

    def attention(self, q, scale, causal=True, window=0):
        """(out, lse, weight, score bound) in 64 bits: weight = sum p |v| / sum p of each value, score bound = the largest
        scale * sum |q k| of each (token, head)."""
        h = q.shape[1]
        g = h // self.kv_heads
        out = torch.zeros(self.n_tok, h, self.hd, dtype=torch.float64)
        mag, lse = out.clone(), torch.zeros(self.n_tok, h, dtype=torch.float64)
        top = lse.clone()
        for b, (a, n) in enumerate(self.seqs):
            t = self.starts[b]
            k, _ = self.rows(self.k_host, b, n)
            v, _ = self.rows(self.v_host, b, n)
            ok = self.seen(b, causal, window)
            for i in range(h):
                qq = q[t:t + a, i].double()
                x = (qq @ k[:, i // g].T * scale).masked_fill(~ok, -math.inf)
                if n:
                    top[t:t + a, i] = (qq.abs() @ k[:, i // g].abs().T * abs(scale)).amax(1)
                lse[t:t + a, i] = torch.logsumexp(x, 1) if n else -math.inf
                p = torch.nan_to_num(torch.softmax(x, 1)) if n else x
                out[t:t + a, i] = p @ v[:, i // g]
                mag[t:t + a, i] = p @ v[:, i // g].abs()
        return out, lse, mag, top

    def mass(self, q, lse, scale, causal=True, window=0, last_q=0):
        """(sum of weights, its error weight) [seqs][kv_heads][max_kv] in 64 bits; the latter is sum p * (scale sum |q k| +
        |lse|)."""
        h = q.shape[1]
        g = h // self.kv_heads
        got = torch.zeros(len(self.seqs), self.kv_heads, self.max_kv, dtype=torch.float64)
        err = got.clone()
        for b, (a, n) in enumerate(self.seqs):
            t = self.starts[b]
            k, _ = self.rows(self.k_host, b, n)
            ok = self.seen(b, causal, window)
            if last_q:
                ok = ok & (torch.arange(a) >= a - last_q)[:, None]
            for i in range(h):
                qq, ll = q[t:t + a, i].double(), lse[t:t + a, i].double()[:, None]
                x = qq @ k[:, i // g].T * scale
                p = torch.exp(x - ll).masked_fill(~ok, 0.0)
                far = qq.abs() @ k[:, i // g].abs().T * abs(scale) + torch.nan_to_num(ll.abs(), posinf=0.0)
                got[b, i // g, :n] += p.sum(0)
                err[b, i // g, :n] += (p * far).sum(0)
        return got, err


def freqs(p):
    """Angle per position of each pair and the factor on cosine and sine, from a CuqRopeParams, in 64 bits."""
    rot = p.rot_dim
    f = [float(p.theta) ** (-2.0 * j / rot) for j in range(rot // 2)]
    if p.scaling == rt.ROPE_LINEAR:
        return [x / p.factor for x in f], 1.0
    if p.scaling == rt.ROPE_LLAMA3:
        s = [min(1.0, max(0.0, (p.orig_ctx * x / (2 * math.pi) - p.low_freq) / (p.high_freq - p.low_freq))) for x in f]
        return [(1 - r) * x / p.factor + r * x for x, r in zip(f, s)], 1.0
    if p.scaling == rt.ROPE_YARN:
        at = lambda t: rot * math.log(p.orig_ctx / (t * 2 * math.pi)) / (2 * math.log(p.theta))  # noqa: E731
        low, high = max(0, math.floor(at(p.beta_fast))), min(rot - 1, math.ceil(at(p.beta_slow)))
        r = [min(1.0, max(0.0, (j - low) / max(high - low, 0.001))) for j in range(rot // 2)]
        mul = p.attn_factor if p.attn_factor > 0 else 0.1 * math.log(p.factor) + 1.0
        return [x / p.factor * y + x * (1 - y) for x, y in zip(f, r)], mul
    return f, 1.0


def rotate(x, pos, p):
    """x [n][heads][hd] turned by pos [n] in 64 bits, and the error weight mul * (|a| + |b|) of each value."""
    f, mul = freqs(p)
    x = x.double()
    y, w = x.clone(), torch.zeros_like(x)
    rot = p.rot_dim
    angle = pos.double()[:, None, None] * torch.tensor(f, dtype=torch.float64)
    co, si = mul * torch.cos(angle), mul * torch.sin(angle)
    ia, ib = (slice(0, rot, 2), slice(1, rot, 2)) if p.adjacent else (slice(0, rot // 2), slice(rot // 2, rot))
    a, b = x[..., ia], x[..., ib]
    y[..., ia], y[..., ib] = a * co - b * si, a * si + b * co
    w[..., ia] = w[..., ib] = mul * (a.abs() + b.abs())
    return y, w


def evict(mass, n, keep, sink, recent):
    """The kept slots of one (sequence, KV head), from the definition."""
    if n <= keep:
        return list(range(n))
    m = [(-math.inf if math.isnan(x) else x) for x in mass[:n].tolist()]
    nan = [math.isnan(x) for x in mass[:n].tolist()]
    mid = sorted(range(sink, n - recent), key=lambda i: (nan[i], -m[i], i))[: keep - sink - recent]
    return list(range(sink)) + sorted(mid) + list(range(n - recent, n))
