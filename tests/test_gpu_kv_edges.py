"""The paged K/V cache (dtts_kv_*) at the edges of what its calls allow: replays over rows that a trim has freed, chunks
behind trimmed pages, queries and outputs in one buffer, large groups of query heads, very many sequences."""
import pytest
import torch

import dtts
import kv_ref as R
from test_gpu_kv import BF, I4, _stream, attend_case, fill, make, rand, read, rng   # noqa: F401 (_stream: a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF, I4])
@pytest.mark.parametrize("page", [16, 64, 128])
@pytest.mark.parametrize("t", [1, 30])
@pytest.mark.parametrize("window,sinks,served", [(0, 0, False), (300, 20, False), (100, 130, False), (100, 20, True), (60, 0, True)])
def test_a_replay_over_trimmed_rows(dtype, page, t, window, sinks, served):
    """A trim frees what a window of 100 with 20 sinks does not see: a graph captured before it for more than that is
    reported, not answered from pages that are gone; one for as much or less is served."""
    g = rng(71)
    n = 700
    kv = make(page=page, dtype=dtype, n_pages=120)
    s = kv.open()
    k, v = rand(g, n + 2 * t, 2, 128), rand(g, n + 2 * t, 2, 128)
    fill(kv, [s], [(k[:n], v[:n])])
    kd, vd, q = k[n:n + t].cuda(), v[n:n + t].cuda(), rand(g, t, 12, 128)
    qd = q.cuda()
    out = torch.zeros_like(qd)
    kv.extend([s], [t])
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=torch.cuda.current_stream()):
        kv.write(0, kd, vd)
        kv.attend(0, qd, out, window=window, sinks=sinks)
    graph.replay()
    kv.sync()                                              # every row is there yet
    free = kv.free_pages()
    kv.trim(s, 100, 20)
    assert kv.free_pages() >= free + 3                     # pages of 128: rows 128 .. 511
    kd.copy_(k[n + t:])
    vd.copy_(v[n + t:])
    kv.extend([s], [t])
    graph.replay()
    if served:
        kv.sync()
        want, tol = R.attend(q, R.held(k, dtype == I4), R.held(v, dtype == I4), n + t, window, sinks, int4=dtype == I4)
        R.assert_close(out, want, tol)
    else:
        with pytest.raises(dtts.DttsError) as e:
            kv.sync()
        assert e.value.status == dtts.ERR_ARG
    kv.sync()
    del graph
    kv.close()


def test_a_captured_read_of_trimmed_rows_is_reported():
    g = rng(72)
    kv = make(page=16, n_pages=60)
    s = kv.open()
    k, v = rand(g, 400, 2, 128), rand(g, 400, 2, 128)
    fill(kv, [s], [(k, v)])
    ko = torch.zeros(1, 400, 2, 128, device="cuda")
    vo = torch.zeros_like(ko)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=torch.cuda.current_stream()):
        kv.read(0, [s], [0], [400], ko, vo)
    graph.replay()
    kv.sync()
    assert torch.equal(ko[0].cpu().double(), R.held(k, True)) and torch.equal(vo[0].cpu().double(), R.held(v, True))
    kv.trim(s, 100, 20)
    kv.extend([s], [0])                                    # sends the trim's marks
    graph.replay()
    with pytest.raises(dtts.DttsError) as e:
        kv.sync()
    assert e.value.status == dtts.ERR_ARG
    kv.sync()
    del graph
    kv.close()


@pytest.mark.parametrize("dtype", [BF, I4])
@pytest.mark.parametrize("page", [16, 32, 64])
@pytest.mark.parametrize("window,sinks", [(100, 20), (37, 0), (100, 5)])
def test_chunks_behind_trimmed_pages(dtype, page, window, sinks):
    """Calls of one, a few and many tokens after each trim; the freed pages are in use by a sequence of NaN."""
    g = rng(73)
    kv = make(page=page, dtype=dtype, n_pages=60)
    s, other = kv.open(), kv.open()
    k, v = rand(g, 700, 2, 128), rand(g, 700, 2, 128)
    fill(kv, [s], [(k[:410], v[:410])])
    n = 410
    for t in (1, 30, 2, 90, 1):
        before = kv.free_pages()
        kv.trim(s, 100, 20)
        rows = min((kv.free_pages() - before) * page, 4096 - kv.length(other))
        if rows:
            fill(kv, [other], [(torch.full((rows, 2, 128), float("nan")).bfloat16(),) * 2])
        fill(kv, [s], [(k[n:n + t], v[n:n + t])])
        q = rand(g, t, 12, 128)
        out = torch.empty(t, 12, 128, dtype=torch.bfloat16, device="cuda")
        kv.attend(0, q.cuda(), out, window=window, sinks=sinks)
        kv.sync()
        n += t
        want, tol = R.attend(q, R.held(k[:n], dtype == I4), R.held(v[:n], dtype == I4), n - t, window, sinks, int4=dtype == I4)
        R.assert_close(out, want, tol, f"{t} tokens at {n - t}")
    kv.close()


@pytest.mark.parametrize("dtype", [BF, I4])
@pytest.mark.parametrize("D,Hq,H", [(128, 12, 2), (64, 4, 2)])
def test_outputs_in_place_of_queries(dtype, D, Hq, H):
    """out may be q: steps in one part and in many, prompts, with rows that are recomputed for a NaN they do not see."""
    g = rng(74)
    lens, news = [3000, 40, 200, 70], [1, 2, 150, 70]
    kv = make(H=H, D=D, dtype=dtype, n_pages=80)
    seqs = [kv.open() for _ in lens]
    rows = [(rand(g, n, H, D), rand(g, n, H, D)) for n in lens]
    for b, j in ((0, 5), (2, 120), (3, 69)):
        rows[b][0][j, 0, 3] = rows[b][1][j, :, 7] = float("nan")
    fill(kv, seqs, [(k[:n - t], v[:n - t]) for (k, v), n, t in zip(rows, lens, news)])
    fill(kv, seqs, [(k[n - t:], v[n - t:]) for (k, v), n, t in zip(rows, lens, news)])
    q = rand(g, sum(news), Hq, D)
    x = q.cuda()
    kv.attend(0, x, x, window=2000, sinks=0)
    kv.sync()
    row = 0
    for b, (n, t) in enumerate(zip(lens, news)):
        want, tol = R.attend(q[row:row + t], R.held(rows[b][0], dtype == I4), R.held(rows[b][1], dtype == I4), n - t, 2000, 0,
                             int4=dtype == I4)
        got = x[row:row + t].cpu()
        assert torch.equal(torch.isnan(got), torch.isnan(want)), f"sequence {b}"
        ok = torch.isfinite(want)
        R.assert_close(torch.where(ok, got.double(), 0), torch.where(ok, want, 0), torch.where(ok, tol, 1e-30), f"sequence {b}")
        row += t
    kv.close()


@pytest.mark.parametrize("dtype", [BF, I4])
@pytest.mark.parametrize("D,Hq,H", [(128, 128, 1), (64, 200, 2), (128, 51, 3), (64, 7, 7)])
def test_large_and_odd_groups(dtype, D, Hq, H):
    attend_case(dtype, D, Hq, H, 32, [1, 70, 150], [1, 3, 1])
    attend_case(dtype, D, Hq, H, 64, [90], [5], window=33, sinks=2)


@pytest.mark.parametrize("dtype", [BF, I4])
def test_very_many_sequences(dtype):
    """More units than the workspace has counters for: one row each, so the output is its value v.  The softmax's sum is
    within 2^-22 of 1 (the exponential of a product's rounding), which a bf16 v does not show; a 4-bit one, of up to 11
    bits, can lie on the border of two bf16 numbers and go to either, half a step or 2^-8 away."""
    g = rng(75)
    n = 33000
    kv = make(H=2, D=64, page=16, dtype=dtype, n_pages=n, max_seqs=n, max_tokens=16)
    seqs = [kv.open() for _ in range(300)]
    seqs += kv.fork(seqs[0], n - 300)
    k, v = rand(g, n, 2, 64), rand(g, n, 2, 64)
    fill(kv, seqs, [(k[i:i + 1], v[i:i + 1]) for i in range(n)])
    out = torch.empty(n, 4, 64, dtype=torch.bfloat16, device="cuda")
    kv.attend(0, rand(g, n, 4, 64).cuda(), out)
    kv.sync()
    want = R.held(v, dtype == I4).repeat_interleave(2, 1)
    if dtype == BF:
        assert torch.equal(out.cpu().double(), want)
    R.assert_close(out, want, want.abs() * (2.0 ** -8 + 2.0 ** -21))
    with pytest.raises(dtts.DttsError) as e:
        kv.open()
    assert e.value.status == dtts.ERR_OOM
    kv.close()


def grow_and_check(kv, seed, dtype, synced):
    """A prompt, steps, a fork that grows and a compaction; synced(): waits for the cache's stream."""
    g = rng(seed)
    s = kv.open()
    k, v = rand(g, 240, 2, 128), rand(g, 240, 2, 128)
    n = 0
    for t in (200, 1, 1, 17, 1):
        kd, vd, q = k[n:n + t].cuda(), v[n:n + t].cuda(), rand(g, t, 12, 128)
        qd, out = q.cuda(), torch.empty(t, 12, 128, dtype=torch.bfloat16, device="cuda")
        torch.cuda.synchronize()
        kv.extend([s], [t])
        kv.write(0, kd, vd)
        kv.attend(0, qd, out)
        synced()
        n += t
        want, tol = R.attend(q, R.held(k[:n], dtype == I4), R.held(v[:n], dtype == I4), n - t, int4=dtype == I4)
        R.assert_close(out, want, tol, f"{t} tokens at {n - t}")
    (f,) = kv.fork(s)
    kv.extend([f], [1])
    keep = list(range(0, n, 3))
    kv.compact(s, keep)
    ko = torch.zeros(1, len(keep), 2, 128, device="cuda")
    vo = torch.zeros_like(ko)
    torch.cuda.synchronize()
    kv.read(0, [s], [0], [len(keep)], ko, vo)
    synced()
    assert torch.equal(ko[0].cpu().double(), R.held(k[keep], dtype == I4))
    assert torch.equal(vo[0].cpu().double(), R.held(v[keep], dtype == I4))
    kv.close_seqs([s, f])


@pytest.mark.parametrize("stream", [None, 1, 2])
def test_the_caches_own_the_legacy_and_the_per_thread_stream(stream):
    for dtype in (BF, I4):
        kv = make(dtype=dtype, page=32)
        kv.set_stream(stream)
        grow_and_check(kv, 76, dtype, kv.sync)
        kv.close()


def test_caches_in_several_threads():
    """Each with its own cache, on its own stream, at the same time."""
    import threading
    failed = []

    def work(seed, dtype):
        try:
            kv = dtts.KVCache(1, 2, 128, 64, 4, 4096, page_tokens=32, dtype=dtype)
            for i in range(5):
                grow_and_check(kv, seed + i, dtype, kv.sync)
            kv.close()
        except BaseException as e:   # noqa: BLE001 (reported below)
            failed.append(e)

    threads = [threading.Thread(target=work, args=(80 + 10 * i, BF if i % 2 else I4)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed


@pytest.mark.parametrize("end,rows", [("truncate", 16), ("trim", 63), ("close", 63), ("compact", 32)])
def test_a_replay_behind_the_end_of_its_batch_spares_the_pages_of_others(end, rows):
    """The header forbids it, and the library cannot see it: but pages that have gone to another sequence since stay as
    that one wrote them."""
    g = rng(91)
    kv = make(page=16, n_pages=9, dtype=BF)
    a, b = kv.open(), kv.open()
    k, v = rand(g, 64, 2, 128), rand(g, 64, 2, 128)
    fill(kv, [b], [(k, v)])
    fill(kv, [a], [(rand(g, 48, 2, 128), rand(g, 48, 2, 128))])
    x = torch.full((1, 2, 128), 9.0, dtype=torch.bfloat16, device="cuda")
    kv.extend([a], [1])                                    # a row on a page of its own
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=torch.cuda.current_stream()):
        kv.write(0, x, x)
    graph.replay()
    free = kv.free_pages()
    if end == "truncate":
        kv.truncate(a, 48)
    elif end == "trim":
        kv.extend([a], [15])                               # the row's page is full and out of the window
        kv.trim(a, 1)
    elif end == "close":
        kv.close_seqs([a])
    else:
        kv.compact(a, list(range(32)))
    assert kv.free_pages() > free
    keep = list(range(1, 1 + rows))
    kv.compact(b, keep)                                    # takes the freed pages, the lowest first
    graph.replay()
    gk, gv = read(kv, b, 0, len(keep))
    assert torch.equal(gk[0].double(), k[keep].double()) and torch.equal(gv[0].double(), v[keep].double())
    kv.close()
