"""The paged K/V cache's operators: what is timed, in plain form and through the library.

Three operators of the cache that serves the LLM decoder's streams:

  attend   attention of the newest tokens of a ragged batch over its cache pages (bf16 or 4-bit rows, grouped
           heads, causal, optionally a sliding window with a few first rows that stay visible)
  store    new rows of K and V into the pages (rounded to 4 bits where the cache holds 4 bits) and back
  branch / compact
           page work: forks of one sequence with the copy of the page they share at the tail, and keeping a
           chosen subset of a sequence's rows, repacked densely

A 4-bit row holds, for every 32 consecutive values x (bf16) of a token's head, one scale
s = clamp(bf16(max|x| / 7), 2^-14, 9344) and the integers c = clamp(round_half_even(x / s), -7, 7); the value it
stands for is c s.  x / s lies either exactly on a rounding border or at least 2^-13 of its size away from it (8-bit
significands on both sides), so c is the same in 32 and in 64 bits."""
import math
import os
import random
import sys

import numpy as np
import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
GROUP = 32


def listed():
    return [
        # one stream a few tokens after its start: latency of the smallest call
        dict(name="attend_first_tokens", op="attend", dtype="int4", seqs=1, len_min=48, len_max=48, new=1,
             heads=12, kv_heads=2, dim=128, page=64, window=0, sinks=0),
        # the benchmark's LLM batch: 64 streams stepping together, ragged prompts up to 512 tokens
        dict(name="attend_batch_step", op="attend", dtype="int4", seqs=64, len_min=65, len_max=512, new=1,
             heads=12, kv_heads=2, dim=128, page=64, window=0, sinks=0),
        # long contexts up to the engine's limit of 32768 tokens
        dict(name="attend_long_step", op="attend", dtype="int4", seqs=32, len_min=4097, len_max=32768, new=1,
             heads=12, kv_heads=2, dim=128, page=64, window=0, sinks=0),
        # the same step where the cache is kept in bf16
        dict(name="attend_bf16_step", op="attend", dtype="bf16", seqs=64, len_min=1000, len_max=8191, new=1,
             heads=12, kv_heads=2, dim=128, page=64, window=0, sinks=0),
        # long-form narration: a window of 1024 tokens and 4 first tokens that stay visible
        dict(name="attend_window_step", op="attend", dtype="int4", seqs=64, len_min=1500, len_max=12000, new=1,
             heads=12, kv_heads=2, dim=128, page=64, window=1024, sinks=4),
        # the PatchEncoder's geometry (16 heads of 64, two tokens per patch), small pages
        dict(name="attend_patch_step", op="attend", dtype="bf16", seqs=32, len_min=60, len_max=500, new=2,
             heads=16, kv_heads=16, dim=64, page=16, window=0, sinks=0),
        # prompts of four streams at once, each over its own rows
        dict(name="attend_prefill", op="attend", dtype="int4", seqs=4, len_min=1501, len_max=2047, new=0,
             heads=12, kv_heads=2, dim=128, page=64, window=0, sinks=0),
        # a chunk of a long prompt behind a window, cache in bf16
        dict(name="attend_chunk_window", op="attend", dtype="bf16", seqs=2, len_min=6001, len_max=9000, new=512,
             heads=12, kv_heads=2, dim=128, page=32, window=4096, sinks=64),
        # one token for each of 8 streams, written and read back
        dict(name="store_step", op="store", dtype="int4", seqs=8, len_min=100, len_max=900, new=1,
             heads=12, kv_heads=2, dim=128, page=64, window=0, sinks=0),
        # four prompts, written and read back
        dict(name="store_prefill", op="store", dtype="int4", seqs=4, len_min=5001, len_max=8000, new=0,
             heads=12, kv_heads=2, dim=128, page=64, window=0, sinks=0),
        # a voice prompt continued by 16 streams: forks, the copies of the shared last page, and their release
        dict(name="branch_prompt", op="branch", dtype="int4", seqs=16, len_min=1000, len_max=1000, new=1,
             heads=12, kv_heads=2, dim=128, page=64, window=0, sinks=0, layers=28),
        # half of a long stream's rows dropped, the rest repacked
        dict(name="compact_half", op="compact", dtype="bf16", seqs=1, len_min=6001, len_max=6001, new=0,
             heads=12, kv_heads=2, dim=128, page=64, window=0, sinks=0, layers=28),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "attend", "store", "branch", "compact"])
    heads, kv_heads, dim = rng.choice([(12, 2, 128), (12, 2, 128), (16, 16, 64), (16, 4, 64), (8, 8, 128), (32, 2, 128)])
    c = dict(op=op, dtype=rng.choice(["int4", "int4", "bf16"]), heads=heads, kv_heads=kv_heads, dim=dim,
             page=rng.choice([16, 32, 64, 128]), window=0, sinks=0)
    if op == "attend":
        if rng.random() < 0.6:                      # a step of one to four tokens
            c["new"] = rng.choice([1, 1, 1, 2, 3, 4])
            c["len_max"] = _log(rng, 16, 32768)
            c["seqs"] = max(1, min(64, _log(rng, 1, 96), 400000 // (c["len_max"] * kv_heads)))
        else:                                       # a prompt or a chunk of one
            c["new"] = _log(rng, 8, 1200)
            c["len_max"] = max(c["new"], min(_log(rng, c["new"], 8000), 60000000 // (c["new"] * heads)))
            c["seqs"] = max(1, min(8, 60000000 // (c["new"] * c["len_max"] * heads)))
        c["len_min"] = max(c["new"], int(c["len_max"] * rng.uniform(0.2, 1.0)))
        if rng.random() < 0.4:
            c["window"] = _log(rng, 1, 4096)
            c["sinks"] = rng.choice([0, 1, 4, 17, 64, 130])
    elif op == "store":
        c["seqs"] = rng.randint(1, 8)
        c["new"] = _log(rng, 1, min(4000, 4000000 // (c["seqs"] * kv_heads * dim)))
        c["len_max"] = c["new"] + _log(rng, 1, 1000)
        c["len_min"] = max(c["new"], int(c["len_max"] * rng.uniform(0.5, 1.0)))
    elif op == "branch":
        c["seqs"] = rng.randint(1, 16)
        c["new"] = rng.randint(1, 5)
        c["len_min"] = c["len_max"] = _log(rng, 2, 3000)
        c["layers"] = rng.randint(1, 14)
    else:
        c["seqs"], c["new"] = 1, 0
        c["len_min"] = c["len_max"] = _log(rng, 8, 3000)
        c["layers"] = rng.randint(1, 14)
    return c


def _lens(case):
    n, lo, hi = case["seqs"], case["len_min"], case["len_max"]
    if n == 1 or case["op"] in ("branch", "compact"):
        return [hi] * (n if case["op"] in ("attend", "store") else 1)
    return [lo + (hi - lo) * ((b * 29) % n) // (n - 1) for b in range(n)]


def _news(case):
    """Newest tokens of each sequence: case["new"], or all of them (0)."""
    return [min(n, case["new"] or n) for n in _lens(case)]


def _keep(case):
    """Rows a compaction keeps: the first four and about half of the others, ascending."""
    n = _lens(case)[0]
    r = random.Random(n)
    return [i for i in range(n) if i < 4 or r.random() < 0.5]


def _first_visible(case, i):
    return max(0, i - case["window"] + 1) if case["window"] else 0


def _inputs(case, seed):
    """K, V rows (bf16) of every sequence and layer and the queries of its newest tokens.  Keys carry a few channels
    four times as large as the others, as rotated keys of a decoder do; values and queries are plain normals."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    H, D, L = case["kv_heads"], case["dim"], case.get("layers", 1)
    tot = sum(_lens(case))
    gain = torch.ones(H, D, device="cuda")
    gain[:, 5::37] = 4.0
    k = torch.empty(L, tot, H, D, device="cuda", dtype=torch.bfloat16)
    v = torch.empty_like(k)
    for l in range(L):
        k[l] = (torch.randn(tot, H, D, device="cuda", generator=g) * gain).bfloat16()
        v[l] = torch.randn(tot, H, D, device="cuda", generator=g).bfloat16()
    q = torch.randn(sum(_news(case)), case["heads"], D, device="cuda", generator=g).bfloat16()
    return k, v, q


def _newest(case):
    """Row indexes (within the concatenated rows) of the newest tokens of all sequences."""
    idx, base = [], 0
    for n, t in zip(_lens(case), _news(case)):
        idx.append(torch.arange(base + n - t, base + n))
        base += n
    return torch.cat(idx).cuda()


# ---------------------------------------------------------------- plain form
def _quantise(x):
    """bf16 [..., D] -> (integers, scales) of the 4-bit rows, in 32 bits."""
    g = x.float().unflatten(-1, (-1, GROUP))
    s = (g.abs().amax(-1, keepdim=True) / 7.0).bfloat16().float().clamp(2.0 ** -14, 9344.0)
    c = torch.round(g / s).clamp(-7, 7)
    return c.to(torch.int8), s


def _dequantise(c, s):
    return (c.float() * s).flatten(-2)


def _held(case, x):
    """Rows as the cache holds them."""
    return _quantise(x) if case["dtype"] == "int4" else x


def _values(case, h):
    return _dequantise(*h) if case["dtype"] == "int4" else h.float()


def _rows(case, h, idx):
    return tuple(t[idx] for t in h) if case["dtype"] == "int4" else h[idx]


def _attend_plain(case, kh, vh, q):
    G, D = case["heads"] // case["kv_heads"], case["dim"]
    out = torch.empty_like(q)
    base = row = 0
    for n, t in zip(_lens(case), _news(case)):
        i0 = n - t
        lo = _first_visible(case, i0)
        sinks = min(case["sinks"], lo)
        j = torch.cat([torch.arange(sinks, device=q.device), torch.arange(lo, n, device=q.device)])
        k = _values(case, _rows(case, kh, base + j))                       # [visible][H][D]
        v = _values(case, _rows(case, vh, base + j))
        qq = q[row:row + t].float().unflatten(1, (-1, G))                  # [t][H][G][D]
        i = torch.arange(i0, n, device=q.device)[:, None]
        ok = j[None] <= i
        if case["window"]:
            ok = ok & ((j[None] > i - case["window"]) | (j[None] < case["sinks"]))
        kk, vv = k.permute(1, 2, 0), v.permute(1, 0, 2)                    # [H][D][n], [H][n][D]
        for a in range(0, t, 512):                                         # scores of 512 queries at a time
            x = qq[a:a + 512]
            m = x.shape[0]
            s = torch.matmul(x.permute(1, 0, 2, 3).flatten(1, 2), kk) / math.sqrt(D)   # [H][m G][visible]
            s = s.unflatten(1, (m, G)).masked_fill(~ok[None, a:a + m, None], -math.inf)
            p = torch.exp(s - s.amax(-1, keepdim=True))
            p = p / p.sum(-1, keepdim=True)
            o = torch.matmul(p.flatten(1, 2), vv).unflatten(1, (m, G))     # [H][m][G][D]
            out[row + a:row + a + m] = o.permute(1, 0, 2, 3).flatten(1, 2).to(q.dtype)
        base += n
        row += t
    return out


def _tail(case):
    """First row of a sequence's last page, and its rows."""
    n = _lens(case)[0]
    first = (n - 1) // case["page"] * case["page"]
    return first, n - first


# ---------------------------------------------------------------- the library
def _dtts():
    pkg = os.path.join(ROOT, "dots.tts.cpp_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import dtts
    return dtts


def _stream():
    # the legacy default stream's handle is 1 (0 would name the cache's own stream)
    return torch.cuda.current_stream().cuda_stream or 1


def _cache(case, k, v):
    """A cache that holds the case's rows, its newest tokens being the current batch."""
    d = _dtts()
    lens, news, page = _lens(case), _news(case), case["page"]
    spare = sum((n + page - 1) // page for n in lens) + 2 * case["seqs"] + 8
    kv = d.KVCache(n_layers=case.get("layers", 1), n_kv_heads=case["kv_heads"], head_dim=case["dim"],
                   n_pages=spare + sum((n + page - 1) // page for n in lens), max_seqs=len(lens) + case["seqs"],
                   max_tokens=max(lens) + 8, page_tokens=page,
                   dtype=d.DTYPE_INT4 if case["dtype"] == "int4" else d.DTYPE_BF16)
    kv.set_stream(_stream())
    seqs = [kv.open() for _ in lens]
    old = [n - t for n, t in zip(lens, news)]
    idx_new = _newest(case)
    is_old = torch.ones(sum(lens), dtype=torch.bool, device="cuda")
    is_old[idx_new] = False
    for part, idx in ((old, is_old.nonzero()[:, 0]), (news, idx_new)):
        if not sum(part):
            continue
        kv.extend(seqs, part)
        for l in range(k.shape[0]):
            kv.write(l, k[l][idx], v[l][idx])
    return kv, seqs


def prepare(case, seed):
    k, v, q = _inputs(case, seed)
    st = dict(case=case, q=q)
    idx = _newest(case)
    st["k_new"], st["v_new"] = k[0][idx].contiguous(), v[0][idx].contiguous()
    if own:
        st["kv"], st["seqs"] = _cache(case, k, v)
        st["keep"] = np.asarray(_keep(case), np.int32)
    elif case["op"] == "attend":
        st["k"], st["v"] = _held(case, k[0]), _held(case, v[0])
    elif case["op"] in ("branch", "compact"):
        st["k"], st["v"] = _held(case, k.transpose(0, 1)), _held(case, v.transpose(0, 1))   # row first
        st["keep"] = torch.tensor(_keep(case), device="cuda")
    torch.cuda.synchronize()
    return st


def run(st):
    case = st["case"]
    return _run_own(case, st) if own else _run_plain(case, st)


def _run_plain(case, st):
    if case["op"] == "attend":
        return _attend_plain(case, st["k"], st["v"], st["q"])
    if case["op"] == "store":
        return [_values(case, _held(case, st[n])) for n in ("k_new", "v_new")]
    out = []
    for h in (st["k"], st["v"]):
        if case["op"] == "branch":
            first, n = _tail(case)
            x = _values(case, _rows(case, h, slice(first, first + n)))     # [n][L][H][D]
            out.append(x.transpose(0, 1)[:, None].repeat(1, case["seqs"], 1, 1, 1))
        else:
            x = _values(case, _rows(case, h, st["keep"]))
            out.append(x.transpose(0, 1).to(torch.bfloat16))
    return out


def _run_own(case, st):
    kv, seqs = st["kv"], st["seqs"]
    kv.set_stream(_stream())
    H, D, L = case["kv_heads"], case["dim"], case.get("layers", 1)
    if case["op"] == "attend":
        out = torch.empty_like(st["q"])
        kv.attend(0, st["q"], out, window=case["window"], sinks=case["sinks"])
        return out
    if case["op"] == "store":
        kv.write(0, st["k_new"], st["v_new"])
        k = torch.empty(st["k_new"].shape, device="cuda")
        v = torch.empty_like(k)
        kv.read(0, seqs, [n - t for n, t in zip(_lens(case), _news(case))], _news(case), k, v)
        return [k, v]
    if case["op"] == "branch":
        first, n = _tail(case)
        k = torch.empty(L, case["seqs"], n, H, D, device="cuda")
        v = torch.empty_like(k)
        forks = kv.fork(seqs[0], case["seqs"])
        kv.extend(forks, [case["new"]] * len(forks))
        kv.read(0, forks, [first] * len(forks), [n] * len(forks), k, v, n_layers=L)
        kv.close_seqs(forks)
        return [k, v]
    n = len(st["keep"])
    k = torch.empty(L, n, H, D, device="cuda", dtype=torch.bfloat16)
    v = torch.empty_like(k)
    (s,) = kv.fork(seqs[0], 1)
    kv.compact(s, st["keep"])
    kv.read(0, [s], [0], [n], k, v, n_layers=L)
    kv.close_seqs([s])
    return [k, v]


# ---------------------------------------------------------------- work and the definition in 64 bits
def _row_bytes(case):
    """Bytes of one token's K and V rows as the cache holds them."""
    D = case["dim"]
    return 2 * case["kv_heads"] * (D // 2 + D // GROUP * 2 if case["dtype"] == "int4" else 2 * D)


def work(case):
    H, D, L = case["kv_heads"], case["dim"], case.get("layers", 1)
    lens, news = _lens(case), _news(case)
    raw = sum(news) * 4 * H * D                       # the newest tokens' K and V in bf16
    if case["op"] == "attend":
        rows = pairs = 0
        for n, t in zip(lens, news):
            lo = _first_visible(case, n - t)
            rows += n - lo + min(case["sinks"], lo)
            for i in range(n - t, n):
                f = _first_visible(case, i)
                pairs += i + 1 - f + min(case["sinks"], f)
        return {"bytes": rows * _row_bytes(case) + 4 * sum(news) * case["heads"] * D,
                "flops": 4.0 * D * case["heads"] * pairs}
    if case["op"] == "store":                         # read, written to the pages, read from them, returned in fp32
        return {"bytes": raw + 2 * sum(news) * _row_bytes(case) + 2 * raw, "flops": 6.0 * sum(news) * 2 * H * D}
    if case["op"] == "branch":
        # the shared page's rows copied for all forks but nobody's original, then read back in fp32
        n = _tail(case)[1]
        copies = case["seqs"] if lens[0] % case["page"] else 0
        return {"bytes": L * n * (_row_bytes(case) * (1 + copies + case["seqs"]) + case["seqs"] * 8 * H * D),
                "flops": 2.0 * case["seqs"] * L * n * H * D}
    n = len(_keep(case))
    return {"bytes": L * n * (3 * _row_bytes(case) + 4 * H * D), "flops": 2.0 * L * n * H * D}


def _exact_rows(case, x):
    if case["dtype"] != "int4":
        return x.double()
    x = x.double()
    y = x.reshape(*x.shape[:-1], case["dim"] // GROUP, GROUP)
    top = y.abs().max(-1).values
    scale = (top / 7.0).to(torch.bfloat16).double()
    scale = torch.minimum(torch.maximum(scale, torch.full_like(scale, 2.0 ** -14)), torch.full_like(scale, 9344.0))
    code = (y / scale[..., None]).round()
    code = torch.where(code > 7, torch.full_like(code, 7), torch.where(code < -7, torch.full_like(code, -7), code))
    return (code * scale[..., None]).reshape(x.shape)


def exact(case, seed):
    k, v, q = _inputs(case, seed)
    if case["op"] == "store":
        idx = _newest(case)
        return [_exact_rows(case, x[0][idx]) for x in (k, v)]
    if case["op"] == "branch":
        first, n = _tail(case)
        return [_exact_rows(case, x[:, first:first + n])[:, None].expand(-1, case["seqs"], -1, -1, -1) for x in (k, v)]
    if case["op"] == "compact":
        keep = torch.tensor(_keep(case), device="cuda")
        return [_exact_rows(case, x[:, keep]) for x in (k, v)]
    G, D = case["heads"] // case["kv_heads"], case["dim"]
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    base = row = 0
    for n, t in zip(_lens(case), _news(case)):
        kk = _exact_rows(case, k[0, base:base + n])
        vv = _exact_rows(case, v[0, base:base + n])
        key = torch.arange(n, device="cuda")
        for a in range(0, t, 256):
            b = min(t, a + 256)
            pos = torch.arange(n - t + a, n - t + b, device="cuda")
            hidden = key[None, :] > pos[:, None]
            if case["window"]:
                hidden |= (key[None, :] <= pos[:, None] - case["window"]) & (key[None, :] >= case["sinks"])
            for h in range(case["heads"]):
                z = (q[row + a:row + b, h].double() @ kk[:, h // G].T) * D ** -0.5
                z[hidden] = float("-inf")
                w = torch.softmax(z, -1)
                out[row + a:row + b, h] = w @ vv[:, h // G]
        base += n
        row += t
    return out
