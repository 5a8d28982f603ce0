"""The paged K/V cache (dtts_kv_*) on the GPU against its definitions in 64 bits (kv_ref)."""
import numpy as np
import pytest
import torch

import dtts
import kv_ref as R

pytestmark = pytest.mark.gpu

BF, I4 = dtts.DTYPE_BF16, dtts.DTYPE_INT4


@pytest.fixture(autouse=True)
def _stream(dtts_mod):
    """Tests run on a stream of their own; caches are put on it by make()."""
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        yield s
    torch.cuda.synchronize()


def rng(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def rand(g, *shape):
    return torch.randn(*shape, generator=g).to(torch.bfloat16)


def make(H=2, D=128, page=64, dtype=I4, layers=1, n_pages=64, max_seqs=16, max_tokens=4096):
    kv = dtts.KVCache(layers, H, D, n_pages, max_seqs, max_tokens, page_tokens=page, dtype=dtype)
    kv.set_stream(torch.cuda.current_stream().cuda_stream)
    return kv


def fill(kv, seqs, rows, layer=0):
    """Appends rows[b] = (k, v) (CPU bf16 [n][H][D]) to the sequences, as one batch."""
    kv.extend(seqs, [len(k) for k, _ in rows])
    kv.write(layer, torch.cat([k for k, _ in rows]).cuda(), torch.cat([v for _, v in rows]).cuda())


def read(kv, seq, first, n, layer=0, n_layers=1, dtype=torch.float32):
    k = torch.empty(n_layers, n, kv.n_kv_heads, kv.head_dim, dtype=dtype, device="cuda")
    v = torch.empty_like(k)
    kv.read(layer, [seq], [first], [n], k, v, n_layers=n_layers)
    torch.cuda.synchronize()
    return k.cpu(), v.cpu()


# ---------------------------------------------------------------- rows
@pytest.mark.parametrize("dtype", [BF, I4])
@pytest.mark.parametrize("D,H,page", [(128, 2, 64), (64, 16, 16), (128, 1, 128), (64, 3, 32)])
def test_rows_are_held_exactly(dtype, D, H, page):
    g = rng(1)
    kv = make(H=H, D=D, page=page, dtype=dtype)
    s = [kv.open(), kv.open()]
    want = [[], []]
    for step in ([5, 0], [1, 70], [3, 131], [129, 1]):   # pages start, continue and end inside a batch
        rows = [(rand(g, n, H, D), rand(g, n, H, D) * 3) for n in step]
        fill(kv, s, rows)
        for b in range(2):
            want[b].append(rows[b])
    for b in range(2):
        n = kv.length(s[b])
        k, v = read(kv, s[b], 0, n)
        for got, at in ((k, 0), (v, 1)):
            x = R.held(torch.cat([w[at] for w in want[b]]), dtype == I4)
            assert torch.equal(got[0].double(), x)
        k2, _ = read(kv, s[b], 2, n - 3, dtype=torch.bfloat16)
        assert torch.equal(k2[0], k[0, 2:n - 1].to(torch.bfloat16))
    kv.close()


def test_int4_borders_and_ranges():
    """Exact ties, the clamped scales, saturation, zeros, subnormals and non-finite groups."""
    kv = make()
    x = torch.zeros(12, 2, 128)
    x[0] = torch.arange(128) % 15 - 7                       # s = 1: integers
    x[1] = (torch.arange(128) % 15 - 7) * 0.5               # s = 0.5
    x[2, :, ::32] = 7.0                                     # s = 1: ties at every half
    x[2, :, 1::32], x[2, :, 2::32], x[2, :, 3::32], x[2, :, 4::32] = 0.5, 1.5, -2.5, -0.5
    x[3] = 1e-6                                             # below the smallest scale
    x[4] = 3e5                                              # above the largest
    x[4, :, 7] = -3.3e38
    x[5] = torch.linspace(-65408, 65408, 128)
    x[6] = 2e-39                                            # bf16 subnormals
    x[7, 0, 3] = float("nan")
    x[8, 1, 40] = float("inf")
    x[9, 0, 100] = float("-inf")
    x[10] = torch.linspace(-1, 1, 128) ** 3
    k = x.to(torch.bfloat16)
    s = kv.open()
    fill(kv, [s], [(k, k.flip(2))])
    got_k, got_v = read(kv, s, 0, 12)
    assert torch.equal(torch.nan_to_num(got_k[0].double(), nan=1e9), torch.nan_to_num(R.held(k, True), nan=1e9))
    assert torch.equal(torch.nan_to_num(got_v[0].double(), nan=1e9), torch.nan_to_num(R.held(k.flip(2), True), nan=1e9))
    kv.close()


def test_rows_from_strided_tensors():
    """k and v inside a fused projection, head-major, and reversed layers of one buffer."""
    g = rng(2)
    kv = make(H=2, D=128, dtype=BF, layers=2)
    s = kv.open()
    qkv = rand(g, 37, 16, 128).cuda()
    hm = rand(g, 2, 37, 128).cuda()
    kv.extend([s], [37])
    kv.write(0, qkv[:, 12:14], qkv[:, 14:16])
    kv.write(1, hm.transpose(0, 1), qkv[:, 3:13:6][:, :2])
    k, v = read(kv, s, 0, 37, n_layers=2, dtype=torch.bfloat16)
    assert torch.equal(k[0], qkv[:, 12:14].cpu()) and torch.equal(v[0], qkv[:, 14:16].cpu())
    assert torch.equal(k[1], hm.transpose(0, 1).cpu()) and torch.equal(v[1], qkv[:, [3, 9]].cpu())
    kv.close()


# ---------------------------------------------------------------- attention
def attend_case(dtype, D, Hq, H, page, lens, news, window=0, sinks=0, seed=3, scale=None, k_gain=1.0, bad_rows=()):
    """Fills the sequences, attends with their newest tokens and compares."""
    g = rng(seed)
    kv = make(H=H, D=D, page=page, dtype=dtype, n_pages=sum(n // page + 2 for n in lens), max_seqs=len(lens) + 1,
              max_tokens=max(lens) + 1)
    seqs = [kv.open() for _ in lens]
    rows = [(rand(g, n, H, D) * k_gain, rand(g, n, H, D)) for n in lens]
    for b, j, value in bad_rows:
        rows[b][0][j] = value
        rows[b][1][j] = value
    fill(kv, seqs, [(k[:n - t], v[:n - t]) for (k, v), n, t in zip(rows, lens, news)])
    fill(kv, seqs, [(k[n - t:], v[n - t:]) for (k, v), n, t in zip(rows, lens, news)])
    q = rand(g, sum(news), Hq, D)
    out = torch.full((sum(news) + 2, Hq, D), 7.0, dtype=torch.bfloat16, device="cuda")
    kv.attend(0, q.cuda(), out[1:-1], scale=scale, window=window, sinks=sinks)
    again = torch.empty_like(out[1:-1])
    kv.attend(0, q.cuda(), again, scale=scale, window=window, sinks=sinks)
    torch.cuda.synchronize()
    kv.sync()
    assert torch.equal(out[1:-1].view(torch.int16), again.view(torch.int16)), "two calls differ"
    assert (out[0] == 7).all() and (out[-1] == 7).all(), "rows around the batch were written"
    row = 1
    for b, (n, t) in enumerate(zip(lens, news)):
        want, tol = R.attend(q[row - 1:row - 1 + t], R.held(rows[b][0], dtype == I4), R.held(rows[b][1], dtype == I4),
                             n - t, window, sinks, scale, dtype == I4)
        R.assert_close(out[row:row + t], want, tol, f"sequence {b} of {n} rows, {t} new")
        row += t
    kv.close()


GEOM = [(128, 12, 2, 64), (64, 16, 16, 16), (128, 8, 8, 32), (64, 16, 4, 128), (128, 32, 2, 64), (64, 3, 1, 32)]


@pytest.mark.parametrize("dtype", [BF, I4])
@pytest.mark.parametrize("D,Hq,H,page", GEOM)
def test_step(dtype, D, Hq, H, page):
    attend_case(dtype, D, Hq, H, page, [1, 15, 16, 17, 63, 64, 65, 200, 517], [1] * 9)


@pytest.mark.parametrize("dtype", [BF, I4])
@pytest.mark.parametrize("D,Hq,H,page", GEOM)
def test_few_tokens(dtype, D, Hq, H, page):
    attend_case(dtype, D, Hq, H, page, [2, 40, 129, 300, 7], [2, 2, 2, 1, 0])


@pytest.mark.parametrize("dtype", [BF, I4])
@pytest.mark.parametrize("window,sinks", [(1, 0), (5, 0), (16, 1), (64, 4), (100, 17), (130, 64), (33, 200), (4000, 3)])
def test_step_window_and_sinks(dtype, window, sinks):
    attend_case(dtype, 128, 12, 2, 64, [1, 3, 64, 130, 333, 700], [1, 1, 1, 1, 1, 1], window, sinks)
    attend_case(dtype, 64, 4, 2, 16, [2, 64, 131, 400], [2, 2, 2, 2], window, sinks)


@pytest.mark.parametrize("dtype", [BF, I4])
def test_step_long_and_split(dtype):
    """Key ranges split over many CTAs and joined, beside short ones."""
    attend_case(dtype, 128, 12, 2, 64, [5000, 12, 2049], [1, 1, 1])
    attend_case(dtype, 64, 8, 8, 16, [3001], [1], window=2500, sinks=5)


@pytest.mark.parametrize("dtype", [BF, I4])
@pytest.mark.parametrize("D,Hq,H,page", GEOM)
def test_prompt(dtype, D, Hq, H, page):
    attend_case(dtype, D, Hq, H, page, [3, 64, 129, 150], [3, 64, 100, 150])


@pytest.mark.parametrize("dtype", [BF, I4])
@pytest.mark.parametrize("window,sinks", [(1, 0), (40, 3), (64, 64), (100, 70), (300, 5)])
def test_prompt_window_and_sinks(dtype, window, sinks):
    attend_case(dtype, 128, 12, 2, 32, [90, 333], [90, 60], window, sinks)
    attend_case(dtype, 64, 4, 4, 16, [300], [140], window, sinks)


@pytest.mark.parametrize("dtype", [BF, I4])
def test_steps_and_prompts_in_one_batch(dtype):
    attend_case(dtype, 128, 12, 2, 64, [100, 70, 500, 33, 1], [1, 70, 2, 5, 1])


@pytest.mark.parametrize("dtype", [BF, I4])
def test_scores_of_any_size(dtype):
    """Sharp softmaxes (one key takes all) and flat ones; a scale of its own."""
    attend_case(dtype, 128, 12, 2, 64, [300, 40], [1, 40], scale=1.0)
    attend_case(dtype, 128, 12, 2, 64, [300, 40], [1, 40], scale=1e-4)
    attend_case(dtype, 64, 4, 4, 32, [200], [1], k_gain=50.0)


# ---------------------------------------------------------------- non-finite values
@pytest.mark.parametrize("dtype", [BF, I4])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_rows_that_a_query_cannot_see_do_not_reach_it(dtype, value):
    """Non-finite K and V behind the window, between sinks and window, and in later rows of the same prompt."""
    g = rng(11)
    for n, t, window, sinks, bad in ((300, 1, 100, 4, [4, 150, 199]), (300, 2, 100, 70, [70, 197]),
                                     (200, 200, 50, 2, [120]), (150, 150, 0, 0, [149, 77]), (2000, 1, 64, 1, [1, 1900])):
        kv = make(dtype=dtype, n_pages=40)
        s = kv.open()
        k, v, q = rand(g, n, 2, 128), rand(g, n, 2, 128), rand(g, t, 12, 128)
        for j in bad:
            k[j, 0, 5], v[j, 1, 40] = value, value
        fill(kv, [s], [(k[:n - t], v[:n - t])])
        fill(kv, [s], [(k[n - t:], v[n - t:])])
        out = torch.empty(t, 12, 128, dtype=torch.bfloat16, device="cuda")
        kv.attend(0, q.cuda(), out, window=window, sinks=sinks)
        want, tol = R.attend(q, R.held(k, dtype == I4), R.held(v, dtype == I4), n - t, window, sinks, None, dtype == I4)
        got = out.cpu()
        assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{n} rows, {t} new"
        ok = torch.isfinite(want)
        R.assert_close(torch.where(ok, got.double(), 0), torch.where(ok, want, 0), torch.where(ok, tol, 1e-30), "finite rows")
        kv.close()


def test_stale_rows_of_a_reused_page_are_not_read():
    """Pages that held NaN are given to another sequence whose last page they fill only partly."""
    g = rng(12)
    for dtype in (BF, I4):
        kv = make(dtype=dtype, n_pages=3)
        s = kv.open()
        fill(kv, [s], [(torch.full((192, 2, 128), float("nan")).bfloat16(),) * 2])
        kv.close_seqs([s])
        for n in (1, 65, 130):
            s = kv.open()
            k, v, q = rand(g, n, 2, 128), rand(g, n, 2, 128), rand(g, n, 12, 128)
            fill(kv, [s], [(k, v)])
            out = torch.empty(n, 12, 128, dtype=torch.bfloat16, device="cuda")
            kv.attend(0, q.cuda(), out)
            want, tol = R.attend(q, R.held(k, dtype == I4), R.held(v, dtype == I4), 0, int4=dtype == I4)
            R.assert_close(out, want, tol, f"{n} rows")
            kv.close_seqs([s])
        kv.close()


# ---------------------------------------------------------------- pages
@pytest.mark.parametrize("dtype", [BF, I4])
def test_forks_share_pages_until_they_grow(dtype):
    g = rng(13)
    L, n = 3, 150
    kv = make(dtype=dtype, layers=L, n_pages=20)
    s = kv.open()
    base = [(rand(g, n, 2, 128), rand(g, n, 2, 128)) for _ in range(L)]
    kv.extend([s], [n])
    for l in range(L):
        kv.write(l, base[l][0].cuda(), base[l][1].cuda())
    forks = kv.fork(s, 3)
    assert kv.free_pages() == 17 and [kv.length(f) for f in forks] == [n] * 3
    more = [[(rand(g, 2, 2, 128), rand(g, 2, 2, 128)) for _ in range(L)] for _ in range(4)]
    kv.extend([s] + forks, [2] * 4)
    assert kv.free_pages() == 14                       # three copies of the shared last page
    for l in range(L):
        kv.write(l, torch.cat([more[b][l][0] for b in range(4)]).cuda(), torch.cat([more[b][l][1] for b in range(4)]).cuda())
    for b, f in enumerate([s] + forks):
        k, v = read(kv, f, 0, n + 2, n_layers=L)
        for l in range(L):
            assert torch.equal(k[l].double(), R.held(torch.cat([base[l][0], more[b][l][0]]), dtype == I4))
            assert torch.equal(v[l].double(), R.held(torch.cat([base[l][1], more[b][l][1]]), dtype == I4))
    kv.close_seqs([s, forks[1]])
    k, _ = read(kv, forks[0], 0, n, n_layers=L)        # the shared pages outlive the sequence they came from
    assert torch.equal(k[2].double(), R.held(base[2][0], dtype == I4))
    (again,) = kv.fork(forks[2])
    kv.truncate(again, 128)                            # at a page border: growing needs no copy
    free = kv.free_pages()
    kv.extend([again], [1])
    assert kv.free_pages() == free - 1
    kv.close_seqs([forks[0], forks[2], again])
    assert kv.free_pages() == 20
    kv.close()


def test_fork_of_an_empty_sequence_and_many_forks():
    kv = make(n_pages=600, max_seqs=1200, max_tokens=64, page=16)
    s = kv.open()
    assert kv.fork(s, 0) == []
    f = kv.fork(s, 1000)
    kv.extend(f[:500], [3] * 500)
    g = rng(14)
    k, v = rand(g, 1500, 2, 128), rand(g, 1500, 2, 128)
    kv.write(0, k.cuda(), v.cuda())
    ko = torch.empty(1, 1500, 2, 128, device="cuda")
    vo = torch.empty_like(ko)
    kv.read(0, f[:500], [0] * 500, [3] * 500, ko, vo)
    assert torch.equal(ko[0].cpu().double(), R.held(k, True)) and torch.equal(vo[0].cpu().double(), R.held(v, True))
    kv.close_seqs(f)
    assert kv.free_pages() == 600
    kv.close()


@pytest.mark.parametrize("dtype", [BF, I4])
@pytest.mark.parametrize("D,page", [(128, 64), (64, 16), (128, 16), (64, 128)])
def test_compact_keeps_the_listed_rows(dtype, D, page):
    g = rng(15)
    L, n = 2, 333
    kv = make(H=3, D=D, page=page, dtype=dtype, layers=L, n_pages=80)
    s = kv.open()
    k, v = rand(g, L, n, 3, D), rand(g, L, n, 3, D)
    kv.extend([s], [n])
    for l in range(L):
        kv.write(l, k[l].cuda(), v[l].cuda())
    for keep in (list(range(n)), list(range(200)) + list(range(230, n)), [0, 1, 2] + list(range(50, 333, 2)),
                 list(range(7, 19)), [332], []):
        (f,) = kv.fork(s)
        kv.compact(f, keep)
        assert kv.length(f) == len(keep) and kv.position(f) == n
        if keep:
            gk, gv = read(kv, f, 0, len(keep), n_layers=L)
            assert torch.equal(gk.double(), R.held(k[:, keep], dtype == I4))
            assert torch.equal(gv.double(), R.held(v[:, keep], dtype == I4))
        kv.extend([f], [1])                            # grows without touching the rows of the source
        kv.write(0, torch.zeros(1, 3, D, dtype=torch.bfloat16, device="cuda"), torch.zeros(1, 3, D, dtype=torch.bfloat16, device="cuda"))
        gk, _ = read(kv, s, 0, n, n_layers=L)
        assert torch.equal(gk.double(), R.held(k, dtype == I4))
        kv.close_seqs([f])
    kv.close()


@pytest.mark.parametrize("dtype", [BF, I4])
def test_trim_frees_what_no_query_sees(dtype):
    g = rng(16)
    window, sinks, n = 100, 20, 400
    kv = make(dtype=dtype, page=32, n_pages=20)
    s = kv.open()
    k, v = rand(g, n + 30, 2, 128), rand(g, n + 30, 2, 128)
    fill(kv, [s], [(k[:n], v[:n])])
    before = kv.free_pages()
    kv.trim(s, window, sinks)
    # the next token, row 400, sees rows 0..19 and 301..; whole pages in between: rows 32..287, 8 pages
    assert kv.free_pages() == before + 8
    fill(kv, [s], [(k[n:n + 1], v[n:n + 1])])
    q = rand(g, 30, 12, 128)
    out = torch.empty(1, 12, 128, dtype=torch.bfloat16, device="cuda")
    kv.attend(0, q[:1].cuda(), out, window=window, sinks=sinks)
    held = [R.held(x, dtype == I4) for x in (k, v)]
    want, tol = R.attend(q[:1], held[0][:n + 1], held[1][:n + 1], n, window, sinks, int4=dtype == I4)
    R.assert_close(out, want, tol, "step")
    for bad in (dict(window=0), dict(window=200, sinks=20), dict(window=100, sinks=33)):
        with pytest.raises(dtts.DttsError) as e:
            kv.attend(0, q[:1].cuda(), out, **bad)
        assert e.value.status == dtts.ERR_ARG
    kv.attend(0, q[:1].cuda(), out, window=113, sinks=32)     # rows 288 .. 400 and 0 .. 31 are there
    with pytest.raises(dtts.DttsError):
        kv.attend(0, q[:1].cuda(), out, window=114)
    with pytest.raises(dtts.DttsError):
        read(kv, s, 31, 2)
    with pytest.raises(dtts.DttsError):
        kv.compact(s, [0, 32])
    with pytest.raises(dtts.DttsError):
        kv.truncate(s, 100)
    kv.truncate(s, 390)
    kv.truncate(s, 300)
    kv.truncate(s, 32)
    fill(kv, [s], [(k[32:40], v[32:40])])
    kv.attend(0, q[:8].cuda(), torch.empty(8, 12, 128, dtype=torch.bfloat16, device="cuda"))   # nothing freed is left
    gk, _ = read(kv, s, 0, 40)
    assert torch.equal(gk[0].double(), held[0][:40])
    kv.close()


def test_refusals():
    kv = make(n_pages=4, max_seqs=3, max_tokens=300)
    s = kv.open()
    x = torch.zeros(8, 2, 128, dtype=torch.bfloat16, device="cuda")
    q = torch.zeros(8, 12, 128, dtype=torch.bfloat16, device="cuda")

    def refused(status, f, *a, **k):
        with pytest.raises(dtts.DttsError) as e:
            f(*a, **k)
        assert e.value.status == status, e.value

    refused(dtts.ERR_ARG, kv.write, 0, x, x)                       # no batch
    refused(dtts.ERR_ARG, kv.attend, 0, q, q)
    refused(dtts.ERR_OOM, kv.extend, [s], [257])
    refused(dtts.ERR_ARG, kv.extend, [s], [301])
    refused(dtts.ERR_ARG, kv.extend, [s], [-1])
    refused(dtts.ERR_ARG, kv.extend, [s, s], [1, 1])
    refused(dtts.ERR_ARG, kv.extend, [s, 2], [1, 1])
    refused(dtts.ERR_ARG, kv.extend, [], [])
    for bad in (-1, 3, 1 << 30):
        refused(dtts.ERR_ARG, kv.extend, [bad], [1])
        refused(dtts.ERR_ARG, kv.close_seqs, [bad])
        refused(dtts.ERR_ARG, kv.fork, bad)
        refused(dtts.ERR_ARG, kv.truncate, bad, 0)
        refused(dtts.ERR_ARG, kv.trim, bad, 1)
        refused(dtts.ERR_ARG, kv.compact, bad, [])
        refused(dtts.ERR_ARG, kv.length, bad)
    assert kv.length(s) == 0 and kv.free_pages() == 4
    kv.extend([s], [8])
    for layer in (-1, 1):
        refused(dtts.ERR_ARG, kv.write, layer, x, x)
        refused(dtts.ERR_ARG, kv.attend, layer, q, q)
    refused(dtts.ERR_ARG, kv.write, 0, x.flatten()[1:1 + 7 * 256].view(7, 2, 128), x)      # off a 16-byte boundary
    refused(dtts.ERR_ARG, kv.write, 0, torch.zeros(8, 2, 130, dtype=torch.bfloat16, device="cuda")[..., :128], x)
    refused(dtts.ERR_ARG, kv.attend, 0, q[:, :11], q[:, :11])
    refused(dtts.ERR_ARG, kv.attend, 0, q, q, window=-1)
    refused(dtts.ERR_ARG, kv.attend, 0, q, q, sinks=-1)
    for scale in (0.0, -1.0, float("nan"), float("inf"), 1e31):
        refused(dtts.ERR_ARG, kv.attend, 0, q, q, scale=scale)
    f32 = torch.zeros(1, 9, 2, 128, device="cuda")
    refused(dtts.ERR_ARG, kv.read, 0, [s], [0], [9], f32, f32.clone())
    refused(dtts.ERR_ARG, kv.read, 0, [s], [-1], [9], f32, f32.clone())
    refused(dtts.ERR_ARG, kv.read, 1, [s], [0], [9], f32, f32.clone())
    refused(dtts.ERR_ARG, kv.compact, s, [1, 1])
    refused(dtts.ERR_ARG, kv.compact, s, [2, 1])
    refused(dtts.ERR_ARG, kv.compact, s, [7, 8])
    refused(dtts.ERR_ARG, kv.truncate, s, 9)
    refused(dtts.ERR_ARG, kv.trim, s, 0)
    refused(dtts.ERR_ARG, kv.close_seqs, [s, s])
    refused(dtts.ERR_OOM, kv.fork, s, 3)
    (f,) = kv.fork(s)
    kv.extend([s], [1])                                            # copies the shared page
    kv.extend([f], [184])                                          # the pool is full now
    refused(dtts.ERR_OOM, kv.extend, [s], [64])
    refused(dtts.ERR_OOM, kv.compact, f, list(range(1, 192)))
    assert kv.length(s) == 9 and kv.length(f) == 192
    kv.close_seqs([f])
    refused(dtts.ERR_ARG, kv.write, 0, x, x)                       # its batch ended with it
    kv.close()
    big = dtts.KVConfig(1 << 10, 32, 128, 128, 1 << 20, 4, 128, I4)   # petabytes
    import ctypes as C
    h = C.c_void_p()
    assert dtts.lib().dtts_kv_create(C.byref(big), 0, C.byref(h)) == dtts.ERR_OOM and not h.value
    make().close()                                                 # and the next one works


# ---------------------------------------------------------------- streams and graphs
def test_captured_step_follows_the_sequences():
    """write + attend captured once; replays act on the batch that is current, across page borders and after a
    sequence was replaced."""
    g = rng(17)
    for dtype in (BF, I4):
        kv = make(dtype=dtype, n_pages=40)
        a, b = kv.open(), kv.open()
        ka, va = rand(g, 230, 2, 128), rand(g, 230, 2, 128)
        kb, vb = rand(g, 230, 2, 128), rand(g, 230, 2, 128)
        fill(kv, [a, b], [(ka[:60], va[:60]), (kb[:190], vb[:190])])
        kn = torch.zeros(2, 2, 128, dtype=torch.bfloat16, device="cuda")
        vn, q, out = torch.zeros_like(kn), torch.zeros(2, 12, 128, dtype=torch.bfloat16, device="cuda"), torch.zeros(2, 12, 128, dtype=torch.bfloat16, device="cuda")
        kv.extend([a, b], [1, 1])
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=torch.cuda.current_stream()):
            kv.write(0, kn, vn)
            kv.attend(0, q, out, window=150, sinks=2)
            with pytest.raises(dtts.DttsError) as e:
                kv.extend([a, b], [1, 1])
            assert e.value.status == dtts.ERR_UNSUPPORTED
            with pytest.raises(dtts.DttsError):
                kv.fork(a)
            with pytest.raises(dtts.DttsError):
                kv.compact(a, [0])
        la, lb, cb = 60, 190, b
        for i in range(12):
            if i:
                if i == 6:
                    kv.close_seqs([cb])
                    cb, lb = kv.open(), 3
                    fill(kv, [cb], [(kb[:3], vb[:3])])
                kv.extend([a, cb], [1, 1])
            kn.copy_(torch.stack([ka[la], kb[lb]]))
            vn.copy_(torch.stack([va[la], vb[lb]]))
            qq = rand(g, 2, 12, 128)
            q.copy_(qq)
            graph.replay()
            la, lb = la + 1, lb + 1
            for row, k, v, n in ((0, ka, va, la), (1, kb, vb, lb)):
                want, tol = R.attend(qq[row:row + 1], R.held(k[:n], dtype == I4), R.held(v[:n], dtype == I4), n - 1, 150, 2)
                R.assert_close(out[row:row + 1], want, tol, f"replay {i}, row {row}")
        del graph
        kv.close()


def test_work_moves_to_another_stream_in_order():
    g = rng(18)
    kv = make(dtype=I4, n_pages=300, max_tokens=16384)
    s = kv.open()
    n = 12000
    k, v, q = rand(g, n, 2, 128).cuda(), rand(g, n, 2, 128).cuda(), rand(g, 4, 12, 128).cuda()
    out = torch.empty_like(q)
    torch.cuda.synchronize()
    other = torch.cuda.Stream()
    for i in range(3):
        kv.extend([s], [n if i == 0 else 0])
        if i == 0:
            kv.write(0, k, v)
        kv.set_stream(other.cuda_stream if i % 2 == 0 else torch.cuda.current_stream().cuda_stream)
        (f,) = kv.fork(s)
        kv.compact(f, list(range(0, n, 2)))
        kv.extend([f], [1])
        kv.write(0, k[:1], v[:1])
        kv.set_stream(None)
        gk = torch.empty(1, 6001, 2, 128, device="cuda")
        gv = torch.empty_like(gk)
        torch.cuda.synchronize()
        kv.read(0, [f], [0], [6001], gk, gv)
        kv.sync()
        assert torch.equal(gk[0].cpu().double(), R.held(torch.cat([k[::2], k[:1]]).cpu(), True))
        kv.close_seqs([f])
    kv.set_stream(1)                       # the legacy default stream
    kv.extend([s], [0])
    kv.attend(0, q, out)                   # no rows: nothing to do
    kv.close()


def test_strided_queries_and_outputs():
    g = rng(19)
    for t in (1, 30):
        kv = make(dtype=I4)
        s = kv.open()
        k, v = rand(g, 100, 2, 128), rand(g, 100, 2, 128)
        fill(kv, [s], [(k[:100 - t], v[:100 - t])])
        fill(kv, [s], [(k[100 - t:], v[100 - t:])])
        qkv = rand(g, t, 16, 128).cuda()
        out = torch.full((12, t, 136), 5.0, dtype=torch.bfloat16, device="cuda")
        kv.attend(0, qkv[:, :12], out[:, :, :128].transpose(0, 1))
        want, tol = R.attend(qkv[:, :12].cpu(), R.held(k, True), R.held(v, True), 100 - t)
        R.assert_close(out[:, :, :128].transpose(0, 1), want, tol)
        assert (out[:, :, 128:] == 5).all()
        kv.close()


def test_pool_beyond_32_bits():
    """Pages past 4 GiB of the pool: the first 2000 of 2100 pages of 2.6 MB are taken."""
    g = rng(20)
    L, n = 40, 130
    kv = make(dtype=BF, layers=L, n_pages=2100, max_tokens=64 * 2000)
    kv.extend([kv.open()], [64 * 2000])
    s = kv.open()
    k, v, q = rand(g, n, 2, 128), rand(g, n, 2, 128), rand(g, n, 12, 128)
    for l in (0, L - 1):
        for t in (n, 1):
            kv.truncate(s, 0)
            kv.extend([s], [n - t])
            kv.write(l, k[:n - t].cuda(), v[:n - t].cuda())
            kv.extend([s], [t])
            kv.write(l, k[n - t:].cuda(), v[n - t:].cuda())
            out = torch.empty(t, 12, 128, dtype=torch.bfloat16, device="cuda")
            kv.attend(l, q[:t].cuda(), out)
            want, tol = R.attend(q[:t], k.double(), v.double(), n - t, int4=False)
            R.assert_close(out, want, tol, f"layer {l}, {t} new")
    (f,) = kv.fork(s)
    kv.extend([f], [1])
    kv.compact(f, list(range(5, n)))
    got, _ = read(kv, f, 0, n - 5, layer=L - 1)
    assert torch.equal(got[0].double(), k[5:].double())
    kv.close()


@pytest.mark.parametrize("dtype", [BF, I4])
@pytest.mark.parametrize("window,sinks", [(2 ** 31 - 1, 0), (2 ** 31 - 1, 2 ** 31 - 1), (0, 2 ** 31 - 1), (5, 2 ** 31 - 1),
                                          (2 ** 31 - 200, 3)])
def test_windows_and_sinks_beyond_every_row(dtype, window, sinks):
    """Row numbers minus such a window do not fit 32 bits."""
    attend_case(dtype, 128, 12, 2, 64, [90, 333, 200], [90, 150, 1], window, sinks)


def test_a_pending_trim_stays_out_of_a_captured_graph():
    """A trim's marks that were pending at a capture do not come back with every replay of the graph."""
    g = rng(21)
    kv = make(page=16, n_pages=40)
    a, b = kv.open(), kv.open()
    ka, va = rand(g, 40, 2, 128), rand(g, 40, 2, 128)
    fill(kv, [a, b], [(ka[:20], va[:20]), (rand(g, 90, 2, 128), rand(g, 90, 2, 128))])
    kn, vn = ka[20:21].cuda(), va[20:21].cuda()
    q = rand(g, 1, 12, 128).cuda()
    out = torch.empty_like(q)
    kv.extend([a], [1])
    kv.write(0, kn, vn)
    kv.attend(0, q, out)
    kv.trim(b, 8)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=torch.cuda.current_stream()):
        kv.write(0, kn, vn)
        kv.attend(0, q, out)
    kv.close_seqs([b])
    c = kv.open()
    assert c == b                                  # the same table row, other pages
    kc, vc = rand(g, 90, 2, 128), rand(g, 90, 2, 128)
    fill(kv, [c], [(kc, vc)])
    for i in range(21, 24):
        kv.extend([a], [1])
        kn.copy_(ka[i:i + 1])
        vn.copy_(va[i:i + 1])
        graph.replay()
        want, tol = R.attend(q.cpu(), R.held(ka[:i + 1], True), R.held(va[:i + 1], True), i, 0, 0, None, True)
        torch.cuda.synchronize()
        R.assert_close(out, want, tol, f"replay at row {i}")
        k, v = read(kv, c, 0, 90)
        assert torch.equal(k[0].double(), R.held(kc, True)) and torch.equal(v[0].double(), R.held(vc, True))
    qc = rand(g, 1, 12, 128)
    kv.extend([c], [1])
    kv.write(0, kc[:1].cuda(), vc[:1].cuda())
    oc = torch.empty(1, 12, 128, dtype=torch.bfloat16, device="cuda")
    kv.attend(0, qc.cuda(), oc)
    torch.cuda.synchronize()
    kk, vv = torch.cat([kc, kc[:1]]), torch.cat([vc, vc[:1]])
    want, tol = R.attend(qc, R.held(kk, True), R.held(vv, True), 90, 0, 0, None, True)
    R.assert_close(oc, want, tol, "the reopened sequence")
    kv.sync()
    kv.close()


def test_tensors_that_do_not_fit_the_batch_are_refused():
    kv = make(page=16, n_pages=8)
    s = kv.open()
    kv.extend([s], [3])
    ok = torch.zeros(3, 2, 128, dtype=torch.bfloat16, device="cuda")
    q = torch.zeros(3, 12, 128, dtype=torch.bfloat16, device="cuda")
    for rows in (ok[:2], ok[:0]):
        for call in (lambda: kv.write(0, rows, ok), lambda: kv.write(0, ok, rows)):
            with pytest.raises(dtts.DttsError) as e:
                call()
            assert e.value.status == dtts.ERR_ARG
    for bad in (ok.half(), ok.cpu(), ok[:, :1], ok[:, :, ::2], ok.float()):
        with pytest.raises(ValueError):
            kv.write(0, bad, ok)
        with pytest.raises(ValueError):
            kv.write(0, ok, bad)
    for call in (lambda: kv.attend(0, q[:2], torch.empty_like(q)), lambda: kv.attend(0, q, q[:2])):
        with pytest.raises(dtts.DttsError) as e:
            call()
        assert e.value.status == dtts.ERR_ARG
    for bad in (q.half(), q.cpu(), q[:, :, :64]):
        with pytest.raises(ValueError):
            kv.attend(0, bad, torch.empty_like(q))
        with pytest.raises(ValueError):
            kv.attend(0, q, bad)
    kv.write(0, ok, ok)
    out = torch.empty(1, 3, 2, 128, device="cuda")
    for bad in (out.half(), out.int(), out.cpu(), out[:, :2], out.bfloat16()):
        with pytest.raises(ValueError):
            kv.read(0, [s], [0], [3], out, bad)
    kv.read(0, [s], [0], [3], out, out.clone())
    torch.cuda.synchronize()
    kv.close()


@pytest.mark.parametrize("n", [7168, 7200, 24600, 60000])
def test_compact_long_sequences(n):
    """Row lists of one launch and of several, runs and single rows far apart."""
    g = rng(31)
    kv = make(H=1, D=64, page=128, n_pages=1000, max_tokens=60000)
    s = kv.open()
    fill(kv, [s], [(rand(g, n, 1, 64), rand(g, n, 1, 64))])
    k, v = read(kv, s, 0, n)
    half = (torch.rand(n, generator=g) < 0.5).nonzero().flatten().tolist()
    for keep in (half, [5, n - 1], [0, 31, 32, 63, 64, 4097] + list(range(n - 70, n)), list(range(1, n))):
        (f,) = kv.fork(s)
        kv.compact(f, keep)
        gk, gv = read(kv, f, 0, len(keep))
        assert torch.equal(gk, k[:, keep]) and torch.equal(gv, v[:, keep])
        kv.close_seqs([f])
    kv.close()


def test_int4_every_pair_of_significands():
    """Each group's largest value against every bf16 value from a 32nd of it up: all quotients a code is rounded from."""
    top, rest = [], []
    for a in range(128, 256):
        x = torch.cat([torch.arange(128, 256) * 2.0 ** -e for e in range(6)])
        x = x[x <= a]
        x = torch.cat([x, x[:-len(x) % 31]]) if len(x) % 31 else x
        x = x.view(-1, 31) * torch.where(torch.arange(31) % 2 == 0, 1.0, -1.0)
        rest.append(x)
        top.append(torch.full((len(x), 1), float(a)))
    rows = torch.cat([torch.cat(top), torch.cat(rest)], 1)
    rows = torch.cat([rows, rows[:-len(rows) % 8]]).view(-1, 2, 128) / 64
    k = rows.to(torch.bfloat16)
    assert torch.equal(k.float(), rows)
    kv = make(n_pages=20)
    s = kv.open()
    fill(kv, [s], [(k, -k)])
    got_k, got_v = read(kv, s, 0, len(k))
    assert torch.equal(got_k[0].double(), R.held(k, True)) and torch.equal(got_v[0].double(), R.held(-k, True))
    kv.close()


@pytest.mark.parametrize("dtype", [BF, I4])
def test_rows_written_after_a_fork_are_shared(dtype):
    """A fork of a sequence of the current batch sees the batch's rows; a grown one keeps its own copy."""
    g = rng(41)
    kv = make(page=32, dtype=dtype)
    s = kv.open()
    k, v = rand(g, 45, 2, 128), rand(g, 45, 2, 128)
    fill(kv, [s], [(k[:40], v[:40])])
    kv.extend([s], [5])
    f, h = kv.fork(s, 2)
    kv.write(0, k[40:].cuda(), v[40:].cuda())
    k2, v2 = rand(g, 3, 2, 128), rand(g, 3, 2, 128)
    fill(kv, [f], [(k2, v2)])
    for seq, wk, wv in ((s, k, v), (h, k, v), (f, torch.cat([k, k2]), torch.cat([v, v2]))):
        gk, gv = read(kv, seq, 0, len(wk))
        assert torch.equal(gk[0].double(), R.held(wk, dtype == I4)) and torch.equal(gv[0].double(), R.held(wv, dtype == I4))
    kv.close()


@pytest.mark.parametrize("dtype", [BF, I4])
@pytest.mark.parametrize("D,Hq,H,page", [(128, 12, 2, 64), (64, 16, 16, 16), (128, 32, 2, 128)])
def test_step_lengths_around_the_choice_of_parts(dtype, D, Hq, H, page):
    """One part, two, and as many as fit, for one stream and for many."""
    attend_case(dtype, D, Hq, H, page, [1100], [1])
    attend_case(dtype, D, Hq, H, page, [9000], [1])
    attend_case(dtype, D, Hq, H, page, [100 + 31 * i for i in range(40)], [1] * 40)


def replay_of(kv, captured, then, dtype, seed):
    """A graph of write + attend captured for a batch of `captured` new tokens a sequence, replayed for `then`; returns
    what was stored and attended then."""
    g = rng(seed)
    seqs = [kv.open() for _ in range(max(len(captured), len(then)))]
    base = [(rand(g, 20 + 7 * b, 2, 128), rand(g, 20 + 7 * b, 2, 128)) for b in range(len(seqs))]
    fill(kv, seqs, base)
    rows = max(sum(captured), sum(then))
    k, v, q = rand(g, rows, 2, 128), rand(g, rows, 2, 128), rand(g, rows, 12, 128)
    kd, vd, qd = k.cuda(), v.cuda(), q.cuda()
    out = torch.full_like(qd, 7.0)
    kv.extend(seqs[:len(captured)], captured)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=torch.cuda.current_stream()):
        kv.write(0, kd, vd)
        kv.attend(0, qd, out)
    for s, n in zip(seqs, base):
        kv.truncate(s, len(n[0]))
    kv.extend(seqs[:len(then)], then)
    graph.replay()
    torch.cuda.synchronize()
    return seqs, base, k, v, q, out, graph


@pytest.mark.parametrize("dtype", [BF, I4])
@pytest.mark.parametrize("captured,then", [
    ([1, 1, 1], [2, 1, 0]),       # 12 rows a key head where 6 were captured
    ([15, 16], [1, 30]),          # a sequence of few rows where only long ones were
    ([1, 2, 2], [5, 0, 0]),       # and the other way round
    ([40, 40], [60, 20]),         # 360 rows where 256 were
    ([1, 40], [30, 50]),          # more rows than the graph knows
    ([1, 1], [1, 1, 1]), ([40], [40, 1]), ([3, 3], [3, 3, 3])])    # more sequences
def test_a_replay_that_does_not_reach_its_batch_is_reported(dtype, captured, then):
    """Rows that the captured launches do not cover are an error at the next sync, not old output; the cache works on."""
    kv = make(dtype=dtype, n_pages=40)
    seqs, base, k, v, q, out, graph = replay_of(kv, captured, then, dtype, 51)
    with pytest.raises(dtts.DttsError) as e:
        kv.sync()
    assert e.value.status == dtts.ERR_ARG, e.value
    kv.sync()                                          # reported once
    kv.write(0, k.cuda(), v.cuda())                    # the batch is current still: eager calls serve it
    kv.attend(0, q.cuda(), out)
    kv.sync()
    at = 0
    for b, t in enumerate(then):
        n = len(base[b][0]) + t
        kk, vv = torch.cat([base[b][0], k[at:at + t]]), torch.cat([base[b][1], v[at:at + t]])
        want, tol = R.attend(q[at:at + t], R.held(kk, dtype == I4), R.held(vv, dtype == I4), n - t, int4=dtype == I4)
        R.assert_close(out[at:at + t], want, tol, f"sequence {b}")
        at += t
    del graph
    kv.close()


@pytest.mark.parametrize("dtype", [BF, I4])
@pytest.mark.parametrize("news", [[1, 1, 1], [2, 1, 0], [40, 1, 2], [60], [43, 50]])
def test_a_replay_of_the_same_counts_is_served(dtype, news):
    kv = make(dtype=dtype, n_pages=40)
    seqs, base, k, v, q, out, graph = replay_of(kv, news, news, dtype, 52)
    kv.sync()
    at = 0
    for b, t in enumerate(news):
        n = len(base[b][0]) + t
        kk, vv = torch.cat([base[b][0], k[at:at + t]]), torch.cat([base[b][1], v[at:at + t]])
        want, tol = R.attend(q[at:at + t], R.held(kk, dtype == I4), R.held(vv, dtype == I4), n - t, int4=dtype == I4)
        R.assert_close(out[at:at + t], want, tol, f"sequence {b}")
        at += t
    del graph
    kv.close()


@pytest.mark.parametrize("t", [1, 30])
@pytest.mark.parametrize("exponent", [-126, -122, -118, -112, -100])
def test_tiny_queries_with_a_large_scale(t, exponent):
    """Queries near the smallest bf16 numbers, brought back by the scale: 4-bit rows take them as halves after an exact
    scaling, which has to reach half's normal range.  All dims pull the same way, so a rounding of q shows."""
    g = rng(61)
    n = 300
    kv = make(dtype=I4)
    s = kv.open()
    sign = torch.where(torch.rand(2, 128, generator=g) < 0.5, -1.0, 1.0)
    k = (sign * (torch.rand(n, 2, 1, generator=g) * 2 - 1) * 2.0 ** 15).to(torch.bfloat16)
    v = rand(g, n, 2, 128)
    size = 1.0 + torch.randint(0, 128, (t, 12, 1), generator=g) / 128     # 8 significant bits
    q = (sign.repeat_interleave(6, 0) * size * 2.0 ** exponent).to(torch.bfloat16)
    scale = float(np.float32(min(1e30, 2.0 ** (-exponent - 22))))           # scores up to 2 or so
    fill(kv, [s], [(k[:n - t], v[:n - t])])
    fill(kv, [s], [(k[n - t:], v[n - t:])])
    out = torch.empty(t, 12, 128, dtype=torch.bfloat16, device="cuda")
    kv.attend(0, q.cuda(), out, scale=scale)
    kv.sync()
    want, tol = R.attend(q, R.held(k, True), R.held(v, True), n - t, scale=scale)
    R.assert_close(out, want, tol)
    kv.close()


def test_positions_after_a_compaction_and_truncations():
    kv = make(page=16, n_pages=20)
    s = kv.open()
    kv.extend([s], [100])
    kv.compact(s, list(range(10)) + list(range(80, 100)))
    assert (kv.length(s), kv.position(s)) == (30, 100)
    kv.extend([s], [5])
    kv.truncate(s, 32)                     # two of the new tokens are left
    assert (kv.length(s), kv.position(s)) == (32, 102)
    kv.truncate(s, 5)                      # 27 rows fewer, whichever positions they had
    assert (kv.length(s), kv.position(s)) == (5, 75)
    kv.extend([s], [1])
    assert (kv.length(s), kv.position(s)) == (6, 76)
    kv.close()
