"""The operators of serving from a paged KV cache, as they are measured: rotary positions with the append into the
cache, attention of new tokens over it, the attention weight that every cached slot has gathered, and the eviction of
the slots that gathered least.

A cache is two pools [pages][kv_heads][page_size][head_dim]; a batch is a run of sequences whose new tokens lie one
behind the other (`q_start`), each with its cache length after the append (`kv_len`) and its row of page numbers.
"""
import ctypes
import math
import random

import torch

own = False

# Geometries (heads, kv_heads, head_dim): the decoder shapes that the benchmark and the tests of this repository use.
SMALL, HALF, MID, BIG = (9, 3, 64), (14, 2, 64), (12, 2, 128), (32, 8, 128)
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
GGML = {"f32": 0, "f16": 1, "bf16": 30}
SCALING = {"none": 0, "linear": 1, "llama3": 2, "yarn": 3}


def _geo(g):
    return {"heads": g[0], "kv_heads": g[1], "hd": g[2]}


def listed():
    return [
        # One new token of each of 16 requests: rotate, convert, append (fp32 projections into an fp16 cache).
        dict(name="append_decode16_f32", op="append", **_geo(BIG), seqs=16, q=1, kv=1500, ragged=1, tail=0, page=16,
             type="f32", cache="f16", out="f32", rot=128, adjacent=True, scaling="none", theta=5e5, far=0),
        # A whole prompt of 4096 tokens at once, positions scaled for a long context.
        dict(name="append_prompt4096_f16", op="append", **_geo(BIG), seqs=1, q=4096, kv=4096, ragged=0, tail=0,
             page=64, type="f16", cache="f16", out="f16", rot=128, adjacent=False, scaling="llama3", theta=5e5, far=0),
        # Chunks of a ragged batch far into long contexts, half of each head rotated, rows behind the last sequence.
        dict(name="append_ragged_bf16", op="append", **_geo(MID), seqs=7, q=509, kv=9001, ragged=2, tail=3, page=32,
             type="bf16", cache="bf16", out="bf16", rot=64, adjacent=False, scaling="yarn", theta=1e6, far=120000),
        # The smallest call: one token of one request over a short context, fp32 activations.
        dict(name="attn_decode1_f32", op="attention", **_geo(SMALL), seqs=1, q=1, kv=609, ragged=0, tail=0, page=16,
             type="f32", cache="f16", causal=True, window=0),
        # A decode step of 32 requests of different lengths up to 8192.
        dict(name="attn_decode32_bf16", op="attention", **_geo(BIG), seqs=32, q=1, kv=8192, ragged=3, tail=0, page=16,
             type="bf16", cache="bf16", causal=True, window=0),
        # A prompt of 4096 tokens from position 0.
        dict(name="attn_prompt4096_f16", op="attention", **_geo(BIG), seqs=1, q=4096, kv=4096, ragged=0, tail=0,
             page=64, type="f16", cache="f16", causal=True, window=0),
        # The next chunk of a long context.
        dict(name="attn_chunk512_long_bf16", op="attention", **_geo(MID), seqs=1, q=512, kv=32768, ragged=0, tail=0,
             page=128, type="bf16", cache="bf16", causal=True, window=0),
        # Chunks and single tokens mixed, sliding window, pages behind the window given back, fp32 activations.
        dict(name="attn_mixed_window_f32", op="attention", **_geo(HALF), seqs=9, q=301, kv=4099, ragged=4, tail=5,
             page=32, type="f32", cache="f16", causal=True, window=1024),
        # The last 32 queries of long prompts as the window that scores the cache before an eviction.
        dict(name="mass_last32_bf16", op="mass", **_geo(BIG), seqs=4, q=32, kv=16384, ragged=5, tail=0, page=16,
             type="bf16", cache="bf16", causal=True, window=0, last_q=32, decay=0.0),
        # Every query of a 2048-token chunk counts.
        dict(name="mass_chunk2048_f16", op="mass", **_geo(MID), seqs=1, q=2048, kv=4096, ragged=0, tail=0, page=64,
             type="f16", cache="f16", causal=True, window=0, last_q=0, decay=1.0),
        # One request's cache from 4096 to 1024 slots.
        dict(name="evict_4096_to_1024_f16", op="evict", **_geo(BIG), seqs=1, kv=4096, ragged=0, page=64, cache="f16",
             keep=1024, sink=4, recent=64),
        # Sixteen long requests of different lengths, down to 4001 slots each.
        dict(name="evict_ragged16_bf16", op="evict", **_geo(MID), seqs=16, kv=32768, ragged=6, page=32, cache="bf16",
             keep=4001, sink=4, recent=256),
    ]


def _log(rng, a, b):
    return max(a, min(b, int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))))


def draw(rng):
    case = _drawn(rng)
    while _cost(case) > _LARGEST and case["seqs"] > 1:
        case["seqs"] -= 1
    while _cost(case) > _LARGEST:
        case["kv"], case["q"] = case["kv"] // 2, min(case["q"], case["kv"] // 2)
    return case


def _drawn(rng):
    op = rng.choice(["append", "attention", "attention", "mass", "evict"])
    geo = rng.choice([SMALL, HALF, MID, BIG, (8, 8, 64), (16, 4, 128), (8, 1, 128)])
    case = dict(op=op, **_geo(geo), seqs=_log(rng, 1, 24), ragged=rng.randrange(1, 1 << 20), tail=rng.choice([0, 0, 3]),
                page=rng.choice([16, 32, 64, 128]))
    pair = rng.choice([("f32", "f16"), ("f16", "f16"), ("bf16", "bf16")])
    if op == "evict":
        case.pop("tail")
        kv = _log(rng, 64, 32768)
        keep = _log(rng, 16, max(16, kv))
        recent = rng.randrange(0, keep // 2 + 1)
        return dict(case, kv=kv, cache=pair[1], keep=keep, sink=min(4, keep - recent), recent=recent)
    if rng.random() < 0.4:
        q, kv = 1, _log(rng, 16, 16384)  # single tokens
    else:
        case["seqs"] = min(case["seqs"], 6)
        q = _log(rng, 2, 2048)
        kv = max(q, _log(rng, 64, 8192))
    case = dict(case, q=q, kv=kv, type=pair[0], cache=pair[1])
    if op == "append":
        half = geo[2] // 2
        return dict(case, out=pair[0], rot=rng.choice([geo[2], geo[2], half]), adjacent=rng.random() < 0.5,
                    scaling=rng.choice(list(SCALING)), theta=rng.choice([1e4, 5e5, 1e6]), far=rng.choice([0, 0, 250000]))
    window = rng.choice([0, 0, _log(rng, 16, 4096)])
    case = dict(case, causal=window > 0 or rng.random() < 0.8, window=window)
    if op == "mass":
        case = dict(case, last_q=rng.choice([0, 0, 32]), decay=rng.choice([0.0, 0.9, 1.0]))
    return case


def _lens(case):
    """[(new tokens, cache length after them)] of each sequence; the first has the largest, one in a larger ragged
    batch is empty."""
    q, kv, n = case.get("q", 0), case["kv"], case["seqs"]
    if not case["ragged"]:
        return [(q, kv)] * n
    r = random.Random(case["ragged"])
    got = [(q, kv)]
    for i in range(1, n):
        ql = 1 if q == 1 or r.random() < 0.4 else r.randint(1, q) if q else 0
        got.append((0, 0) if n > 4 and i == n // 2 else (ql, max(ql, int(math.exp(r.uniform(math.log(16), math.log(max(17, kv))))))))
    return [(a, min(b, kv)) for a, b in got]


def _visible(case, ql, kl):
    """(query, key) pairs that are visible in one sequence, and the slots that any of its queries sees."""
    w, pairs, first = case["window"], 0, kl
    if not ql:
        return 0, 0
    if not case["causal"]:
        return ql * kl, kl
    for p in range(kl - ql, kl):
        lo = max(0, p + 1 - w) if w else 0
        pairs += p + 1 - lo
        first = min(first, lo)
    return pairs, kl - first


def _freqs(case):
    """Angle per position of each pair, in 64 bits, and the factor on cosine and sine."""
    rot, theta, kind = case["rot"], case["theta"], case["scaling"]
    f = [theta ** (-2.0 * j / rot) for j in range(rot // 2)]
    if kind == "linear":
        return [x / 4.0 for x in f], 1.0
    if kind == "llama3":  # factor 8, low 1, high 4, original context 8192
        got = []
        for x in f:
            turns = 8192.0 * x / (2 * math.pi)
            s = min(1.0, max(0.0, (turns - 1.0) / (4.0 - 1.0)))
            got.append((1 - s) * x / 8.0 + s * x)
        return got, 1.0
    if kind == "yarn":  # factor 4, original context 32768, 32 and 1 turns
        at = lambda turns: rot * math.log(32768 / (turns * 2 * math.pi)) / (2 * math.log(theta))  # noqa: E731
        low, high = max(0, math.floor(at(32.0))), min(rot - 1, math.ceil(at(1.0)))
        ramp = [min(1.0, max(0.0, (j - low) / max(high - low, 0.001))) for j in range(rot // 2)]
        return [x / 4.0 * r + x * (1 - r) for x, r in zip(f, ramp)], 0.1 * math.log(4.0) + 1.0
    return f, 1.0


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    r = random.Random(seed)
    lens = _lens(case)
    h, kvh, hd, page = case["heads"], case["kv_heads"], case["hd"], case["page"]
    ct = TYPES[case["cache"]]
    cols = max(1, -(-case["kv"] // page))
    need = [-(-kl // page) for _, kl in lens]
    n_pages = sum(need) + 3
    ids = list(range(n_pages - 1))  # the last page is nobody's
    r.shuffle(ids)
    table = torch.full((len(lens), cols), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = torch.tensor(ids[at:at + n], dtype=torch.int32)
        at += n
        w = case.get("window", 0)
        if w:  # pages wholly behind every window are given back
            table[b, : max(0, lens[b][1] - lens[b][0] + 1 - w) // page] = -1
    rand = lambda *shape: torch.randn(*shape, device="cuda", generator=g)  # noqa: E731
    k = rand(n_pages, kvh, page, hd).to(ct)
    v = rand(n_pages, kvh, page, hd).to(ct)
    s = {"case": case, "k": k, "v": v, "pages": table.cuda(), "n_pages": n_pages,
         "kv_len": torch.tensor([b for _, b in lens], dtype=torch.int32, device="cuda"), "scale": hd ** -0.5}
    if case["op"] == "evict":
        # gathered attention weight: heavy-tailed, some slots never seen (exact ties at 0)
        m = torch.exp(2.0 * rand(len(lens), kvh, case["kv"])) * (rand(len(lens), kvh, case["kv"]) > -1.0)
        s |= {"mass": m, "kept": torch.full((len(lens), kvh, case["keep"]), -1, dtype=torch.int32, device="cuda"),
              "len": torch.zeros(len(lens), dtype=torch.int32, device="cuda"), "mass_out": torch.zeros_like(m)}
        return s
    starts = [0]
    for a, _ in lens:
        starts.append(starts[-1] + a)
    n = starts[-1] + case["tail"]
    t = TYPES[case["type"]]
    s |= {"q_start": torch.tensor(starts, dtype=torch.int32, device="cuda"), "n_tok": n}
    if case["op"] == "append":
        f, mul = _freqs(case)
        pos = [p + case["far"] for a, b in lens for p in range(b - a, b)] + [0] * case["tail"]
        s |= {"qkv": rand(n, (h + 2 * kvh) * hd).to(t), "positions": torch.tensor(pos, dtype=torch.int32, device="cuda"),
              "freqs": torch.tensor(f, dtype=torch.float64, device="cuda"), "mul": mul,
              "q_out": torch.zeros(n, h, hd, dtype=TYPES[case["out"]], device="cuda")}
        return s
    s["q"] = (1.5 * rand(n, h, hd)).to(t)
    if case["op"] == "attention":
        s |= {"out": torch.zeros(n, h, hd, dtype=t, device="cuda"),
              "lse": torch.zeros(n, h, dtype=torch.float32, device="cuda")}
    else:
        s |= {"mass": torch.rand(len(lens), kvh, case["kv"], device="cuda", generator=g)}
        s["lse"] = _attend(s, True)[1].clone()
    return s


# ------------------------------------------------------------------ plain forms ----


def _dense(s, pool):
    """The cache rows of every sequence as [seqs][kv_heads][slots][hd] in 32 bits; holes hold page 0."""
    x = pool[s["pages"].clamp(0, s["n_pages"] - 1).long()]  # [B, P, H, page, hd]
    b, p, h, n, d = x.shape
    return x.permute(0, 2, 1, 3, 4).reshape(b, h, p * n, d).float()


def _padded(s):
    """(row numbers [seqs][max_q] of the new tokens, n_tok where there is none; their cache slots; slots counted)."""
    c = s["case"]
    start, i = s["q_start"].long(), torch.arange(c["q"], device="cuda")
    ql = start[1:] - start[:-1]
    tok = torch.where(i < ql[:, None], start[:-1, None] + i, s["n_tok"])
    return tok, s["kv_len"].long()[:, None] - ql[:, None] + i, ql


def _mask(s, slot):
    """[seqs][max_q][slots]: whether a query sees a slot."""
    c = s["case"]
    key = torch.arange(s["pages"].shape[1] * c["page"], device="cuda")
    there = ((s["pages"] >= 0) & (s["pages"] < s["n_pages"])).repeat_interleave(c["page"], 1)
    ok = (there & (key < s["kv_len"][:, None]))[:, None, :] & (slot >= 0)[:, :, None]
    if c["causal"]:
        ok = ok & (key <= slot[:, :, None])
        if c["window"]:
            ok = ok & (key > slot[:, :, None] - c["window"])
    return ok


def _scores(s):
    c = s["case"]
    h, kvh, hd = c["heads"], c["kv_heads"], c["hd"]
    tok, slot, ql = _padded(s)
    b, nq = tok.shape
    q = s["q"].float()[tok.clamp(max=max(0, s["n_tok"] - 1))]
    q = q.view(b, nq, kvh, h // kvh, hd).permute(0, 2, 3, 1, 4).reshape(b, kvh, -1, hd)
    x = (q @ _dense(s, s["k"]).transpose(2, 3)).mul_(s["scale"]).view(b, kvh, h // kvh, nq, -1)
    return x, tok, slot, ql


def _attend(s, lse_only=False):
    c = s["case"]
    x, tok, slot, _ = _scores(s)
    x = x.masked_fill_(~_mask(s, slot)[:, None, None], -math.inf)
    b, kvh, g, nq, n = x.shape
    top = x.amax(4, keepdim=True)
    x = x.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = x.sum(4, keepdim=True)
    lse = (top + total.log()).squeeze(4).permute(0, 3, 1, 2).reshape(b, nq, -1)
    flat = tok.reshape(-1)
    all_lse = torch.zeros(s["n_tok"] + 1, c["heads"], device="cuda")
    all_lse[flat] = lse.reshape(-1, c["heads"])
    if lse_only:
        return None, all_lse[:-1]
    o = x.view(b, kvh, g * nq, n) @ _dense(s, s["v"])
    o = o.view(b, kvh, g, nq, -1) / torch.where(total == 0, 1.0, total)
    out = torch.zeros(s["n_tok"] + 1, c["heads"], c["hd"], dtype=s["q"].dtype, device="cuda")
    out[flat] = o.permute(0, 3, 1, 2, 4).reshape(b * nq, c["heads"], c["hd"]).to(out.dtype)
    return out[:-1], all_lse[:-1]


def _weigh(s):
    c = s["case"]
    x, tok, slot, ql = _scores(s)
    seen = _mask(s, slot)
    i = torch.arange(c["q"], device="cuda")
    counts = i < ql[:, None]
    if c["last_q"]:
        counts = counts & (i >= ql[:, None] - c["last_q"])
    seen = seen & counts[:, :, None]
    b, kvh, g, nq, n = x.shape
    lse = s["lse"][tok.clamp(max=max(0, s["n_tok"] - 1))].view(b, nq, kvh, g).permute(0, 2, 3, 1)
    x = x.sub_(lse[..., None]).masked_fill_(~seen[:, None, None], -math.inf).exp_()
    add = x.sum((2, 3))[:, :, : c["kv"]]
    key = torch.arange(c["kv"], device="cuda")
    inside = (key < s["kv_len"][:, None])[:, None]
    s["mass"].copy_(torch.where(inside, c["decay"] * s["mass"] + add, s["mass"]))
    return s["mass"]


def _rows(s, slot, valid):
    """Flat row numbers [seqs][slots][kv_heads] in a pool's [pages * kv_heads * page] rows; None of them for invalid."""
    c = s["case"]
    col = (slot.clamp(min=0) // c["page"]).clamp(max=s["pages"].shape[1] - 1)
    page = s["pages"].long().gather(1, col.reshape(col.shape[0], -1)).view_as(col)
    return page, slot.clamp(min=0) % c["page"], valid & (slot >= 0) & (page >= 0) & (page < s["n_pages"])


def _rotate(s, x):
    c = s["case"]
    rot, half = c["rot"], c["rot"] // 2
    angle = s["positions"].double()[:, None] * s["freqs"]
    co, si = ((f(angle) * s["mul"]).float()[:, None, :] for f in (torch.cos, torch.sin))
    y = x.clone()
    if c["adjacent"]:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        y[..., 0:rot:2], y[..., 1:rot:2] = a * co - b * si, a * si + b * co
    else:
        a, b = x[..., :half], x[..., half:rot]
        y[..., :half], y[..., half:rot] = a * co - b * si, a * si + b * co
    return y


def _append(s):
    c = s["case"]
    h, kvh, hd, n = c["heads"], c["kv_heads"], c["hd"], s["n_tok"]
    q, k, v = (x.float().view(n, -1, hd) for x in s["qkv"].split([h * hd, kvh * hd, kvh * hd], 1))
    used = torch.arange(n, device="cuda") < s["q_start"][-1]
    s["q_out"].copy_(torch.where(used[:, None, None], _rotate(s, q).to(s["q_out"].dtype), s["q_out"]))
    tok, slot, ql = _padded(s)
    valid = tok < n
    page, inside, ok = _rows(s, slot, valid)
    t = tok.clamp(max=n - 1).reshape(-1)
    page, inside, ok = (x.reshape(-1) for x in (page, inside, ok))
    # where there is no row to write, the last page's first row (nobody's) is written over itself
    spare = s["n_pages"] - 1
    to, inside = torch.where(ok, page, spare), torch.where(ok, inside, 0)
    for pool, x in ((s["k"], _rotate(s, k)), (s["v"], v)):
        pool[to, :, inside] = torch.where(ok[:, None, None], x.to(pool.dtype)[t], pool[spare, :, 0])
    return {"q": s["q_out"], "k": s["k"], "v": s["v"]}


def _evict(s):
    c = s["case"]
    b, kvh, kv = s["mass"].shape
    keep, n = c["keep"], s["kv_len"].long()
    key = torch.arange(kv, device="cuda")
    forced = (key < c["sink"]) | (key >= n[:, None] - c["recent"])
    m = torch.where(forced[:, None], math.inf, s["mass"])
    m = torch.where((key < n[:, None])[:, None], m, -math.inf)
    order = torch.sort(m, dim=2, descending=True, stable=True).indices
    order = order[:, :, :keep] if keep <= kv else torch.nn.functional.pad(order, (0, keep - kv), value=kv)
    count = torch.minimum(n, torch.tensor(keep, device="cuda"))
    live = torch.arange(keep, device="cuda") < count[:, None]
    kept = torch.where(live[:, None], order, kv + 1).sort(dim=2).values
    s["kept"].copy_(torch.where(live[:, None], kept, -1))
    s["len"].copy_(count)
    at = kept.clamp(max=kv - 1)
    moved = s["mass"].gather(2, at)
    width = min(keep, kv)
    new = torch.zeros_like(s["mass"])
    new[:, :, :width] = torch.where(live[:, None], moved, 0.0)[:, :, :width]
    s["mass_out"].copy_(torch.where((key < n[:, None])[:, None], new, s["mass_out"]))
    head = torch.arange(kvh, device="cuda")[None, :, None].expand(b, kvh, keep)
    pages = s["pages"].long()
    src = pages.gather(1, (at // c["page"]).view(b, -1)).view(b, kvh, keep)
    to = torch.arange(keep, device="cuda").clamp(max=kv - 1).expand(b, kvh, keep)
    dst = pages.gather(1, (to // c["page"]).reshape(b, -1)).view(b, kvh, keep)
    ok = live[:, None].expand(b, kvh, keep)
    spare = s["n_pages"] - 1  # nobody's: its first row is written over itself where there is nothing to move
    dst, inside = torch.where(ok, dst, spare), torch.where(ok, to % c["page"], 0)
    for pool in (s["k"], s["v"]):
        rows = pool[src.clamp(min=0), head, at % c["page"]]
        pool[dst, head, inside] = torch.where(ok[..., None], rows, pool[spare, head, 0])
    return {"kept": s["kept"], "len": s["len"], "mass": s["mass_out"], "k": s["k"], "v": s["v"]}


# ------------------------------------------------------------- the framework's calls ----


def _handles(s):
    """The descriptors that a program keeps for its cache and its batch."""
    from anedvd_b200 import runtime as rt

    c = s["case"]
    if not rt.load().cuq_ready():  # once in a program
        rt.init(torch.cuda.current_device())
    kv = rt.CuqPagedKv(k=s["k"].data_ptr(), v=s["v"].data_ptr(), type=GGML[c["cache"]], n_pages=s["n_pages"],
                       page_size=c["page"], kv_heads=c["kv_heads"], head_dim=c["hd"], page_stride=0)
    start = s.get("q_start")
    batch = rt.CuqBatch(q_start=None if start is None else start.data_ptr(), kv_len=s["kv_len"].data_ptr(),
                        pages=s["pages"].data_ptr(), n_seqs=c["seqs"], n_tok=s.get("n_tok", 0),
                        pages_stride=s["pages"].shape[1], max_q=c.get("q", 0), max_kv=c["kv"])
    got = {"rt": rt, "lib": rt.load(), "kv": ctypes.byref(kv), "batch": ctypes.byref(batch)}
    if c["op"] == "append":
        p = rt.CuqRopeParams(rot_dim=c["rot"], adjacent=int(c["adjacent"]), theta=c["theta"], scaling=SCALING[c["scaling"]])
        if c["scaling"] == "linear":
            p.factor = 4.0
        elif c["scaling"] == "llama3":
            p.factor, p.low_freq, p.high_freq, p.orig_ctx = 8.0, 1.0, 4.0, 8192
        elif c["scaling"] == "yarn":
            p.factor, p.beta_fast, p.beta_slow, p.orig_ctx = 4.0, 32.0, 1.0, 32768
        got["plan"] = rt.RopePlan(p)
    if c["op"] == "attention":
        need = rt.load().cuq_attention_paged_workspace(got["kv"], got["batch"], c["heads"], GGML[c["type"]])
        got["space"], got["bytes"] = torch.empty(max(1, need), dtype=torch.uint8, device="cuda"), need
    return got


def _own(s):
    c = s["case"]
    if "own" not in s:
        s["own"] = _handles(s)
    o = s["own"]
    lib, check = o["lib"], o["rt"].check
    stream = torch.cuda.current_stream().cuda_stream
    if c["op"] == "append":
        size, row = s["qkv"].element_size(), s["qkv"].shape[1]
        q = s["qkv"].data_ptr()
        k = q + c["heads"] * c["hd"] * size
        check(lib.cuq_rope_append(o["plan"].handle, o["kv"], o["batch"], s["positions"].data_ptr(), s["q_out"].data_ptr(),
                                  c["heads"] * c["hd"], GGML[c["out"]], q, row, k, k + c["kv_heads"] * c["hd"] * size, row,
                                  GGML[c["type"]], c["heads"], stream))
        return {"q": s["q_out"], "k": s["k"], "v": s["v"]}
    if c["op"] == "attention":
        row = c["heads"] * c["hd"]
        check(lib.cuq_attention_paged(o["kv"], o["batch"], s["out"].data_ptr(), row, s["q"].data_ptr(), row,
                                      GGML[c["type"]], s["lse"].data_ptr(), c["heads"], s["scale"], int(c["causal"]),
                                      c["window"], o["space"].data_ptr(), o["bytes"], stream))
        return {"out": s["out"], "lse": s["lse"]}
    if c["op"] == "mass":
        row = c["heads"] * c["hd"]
        check(lib.cuq_attention_mass(o["kv"], o["batch"], s["mass"].data_ptr(), s["mass"].shape[2], s["q"].data_ptr(), row,
                                     GGML[c["type"]], s["lse"].data_ptr(), c["heads"], s["scale"], int(c["causal"]),
                                     c["window"], c["last_q"], c["decay"], stream))
        return {"mass": s["mass"]}
    check(lib.cuq_kv_evict(o["kv"], o["batch"], s["mass"].data_ptr(), s["mass"].shape[2], c["keep"], c["sink"], c["recent"],
                           s["kept"].data_ptr(), s["len"].data_ptr(), s["mass_out"].data_ptr(), s["mass_out"].shape[2],
                           stream))
    return {"kept": s["kept"], "len": s["len"], "mass": s["mass_out"], "k": s["k"], "v": s["v"]}


def run(state):
    if own:
        return _own(state)
    op = state["case"]["op"]
    if op == "append":
        return _append(state)
    if op == "attention":
        out, lse = _attend(state)
        return {"out": out, "lse": lse}
    if op == "mass":
        return {"mass": _weigh(state)}
    return _evict(state)


def work(case):
    lens, h, kvh, hd = _lens(case), case["heads"], case["kv_heads"], case["hd"]
    csize = 2
    if case["op"] == "evict":
        kept = sum(min(b, case["keep"]) for _, b in lens)
        slots = sum(b for _, b in lens)
        return {"bytes": kvh * (slots * 8 + kept * 4) + kept * kvh * hd * csize * 4, "flops": kvh * slots}
    size = {"f32": 4}.get(case["type"], 2)
    toks = sum(a for a, _ in lens)
    if case["op"] == "append":
        return {"bytes": toks * hd * (size * (2 * h + 2 * kvh) + 2 * csize * kvh), "flops": 3 * toks * case["rot"] * (h + kvh)}
    pairs = slots = 0
    for a, b in lens:
        if case["op"] == "mass" and case["last_q"]:
            a = min(a, case["last_q"])
        p, n = _visible(case, a, b)
        pairs, slots = pairs + p, slots + n
    if case["op"] == "attention":
        return {"bytes": slots * kvh * hd * csize * 2 + toks * h * (hd * size * 2 + 4), "flops": 4 * pairs * h * hd}
    used = sum(min(a, case["last_q"]) if case["last_q"] else a for a, _ in lens)
    return {"bytes": slots * kvh * (hd * csize + 8) + used * h * (hd * size + 4), "flops": 2 * pairs * h * hd}


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 50)


_LARGEST = max(_cost(c) for c in listed())


# ------------------------------------------------------------------ from the definition ----


def _slots(s, b, n):
    """Page number and place in the page of slots 0..n-1 of sequence b."""
    i = torch.arange(n, device="cuda")
    return s["pages"][b].long()[i // s["case"]["page"]], i % s["case"]["page"]


def exact(case, seed):
    s = prepare(case, seed)
    lens, h, kvh, hd = _lens(case), case["heads"], case["kv_heads"], case["hd"]
    f64 = dict(dtype=torch.float64, device="cuda")
    if case["op"] == "evict":
        mass = s["mass"].double()
        new = torch.zeros(mass.shape, **f64)
        for b, (_, n) in enumerate(lens):
            for j in range(kvh):
                m = mass[b, j, :n].tolist()
                edge = max(case["sink"], n - case["recent"])
                free = max(0, min(n, case["keep"]) - (n - edge) - min(case["sink"], n))
                best = sorted(range(case["sink"], edge), key=lambda i: (-m[i], i))[:free]
                ids = list(range(min(case["sink"], n))) + sorted(best) + list(range(edge, n))
                ids = ids[: case["keep"]] if n > case["keep"] else list(range(n))
                new[b, j, : len(ids)] = mass[b, j, torch.tensor(ids, dtype=torch.long, device="cuda")]
        return {"kept": None, "len": None, "mass": new, "k": None, "v": None}
    if case["op"] == "append":
        x = s["qkv"].double().view(s["n_tok"], h + 2 * kvh, hd)
        z = x.clone()
        f, mul = _freqs(case)
        at = s["positions"].double()
        for j, w in enumerate(f):
            i0, i1 = (2 * j, 2 * j + 1) if case["adjacent"] else (j, j + case["rot"] // 2)
            co, si = mul * torch.cos(at * w)[:, None], mul * torch.sin(at * w)[:, None]
            z[:, : h + kvh, i0] = x[:, : h + kvh, i0] * co - x[:, : h + kvh, i1] * si
            z[:, : h + kvh, i1] = x[:, : h + kvh, i1] * co + x[:, : h + kvh, i0] * si
        k, v, t = s["k"].double(), s["v"].double(), 0
        q = torch.zeros(s["n_tok"], h, hd, **f64)
        for b, (a, n) in enumerate(lens):
            page, place = (u[n - a:] for u in _slots(s, b, n))
            q[t:t + a] = z[t:t + a, :h]
            k[page, :, place] = z[t:t + a, h:h + kvh]
            v[page, :, place] = z[t:t + a, h + kvh:]
            t += a
        return {"q": q, "k": k, "v": v}
    out, lse = torch.zeros(s["n_tok"], h, hd, **f64), torch.zeros(s["n_tok"], h, **f64)
    mass, t, g = s["mass"].double() if case["op"] == "mass" else None, 0, h // kvh
    for b, (a, n) in enumerate(lens):
        page, place = _slots(s, b, n)
        key = torch.arange(n, device="cuda")
        mine = torch.arange(n - a, n, device="cuda")[:, None]
        ok = (page >= 0).expand(a, n)
        if case["causal"]:
            ok = ok & (key <= mine)
            if case["window"]:
                ok = ok & (key + case["window"] > mine)
        for j in range(kvh):
            rows, vals = s["k"][page, j, place].double(), s["v"][page, j, place].double()
            for i in range(j * g, j * g + g):
                x = (s["q"][t:t + a, i].double() @ rows.T) * s["scale"]
                x = torch.where(ok, x, -math.inf)
                if case["op"] == "attention":
                    lse[t:t + a, i] = torch.logsumexp(x, 1)
                    out[t:t + a, i] = torch.nan_to_num(torch.softmax(x, 1)) @ vals
                else:
                    p = torch.exp(x - s["lse"][t:t + a, i].double()[:, None])
                    p = p[max(0, a - case["last_q"]):] if case["last_q"] else p
                    mass[b, j, :n] = mass[b, j, :n] * (case["decay"] if i == j * g else 1.0) + p.sum(0)
        t += a
    return {"mass": mass} if case["op"] == "mass" else {"out": out, "lse": lse}
