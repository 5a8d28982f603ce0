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
