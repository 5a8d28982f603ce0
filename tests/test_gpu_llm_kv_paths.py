"""The decoder over a paged cache (dtts_llm_extend) on the paths that short batches do not take: more than 256 tokens
in a call, steps whose key ranges are split, and split otherwise as the streams grow, sequences after a compaction, and
step graphs of more shapes than are kept.  Against a decoder in 64 bits with an explicit mask."""
import numpy as np
import pytest
import torch

import dtts
import kv_ref as R
import synth
from helpers import assert_bf16_close, assert_no_worse_than_recipe

pytestmark = pytest.mark.gpu

LAYERS = 2
BF, I4 = dtts.DTYPE_BF16, dtts.DTYPE_INT4


@pytest.fixture(scope="module")
def weights():
    return synth.llm_weights(3, n_layers=LAYERS)


@pytest.fixture(scope="module")
def wide(weights):
    return {k: torch.from_numpy(np.ascontiguousarray(v)).double().cuda() for k, v in weights.items() if k.startswith("llm.model.")}


@pytest.fixture(scope="module")
def llm(weights):
    e = dtts.LLM(weights, n_layers=LAYERS, max_batch=4, max_seq=2048)
    yield e
    e.close()


def emb_of(name, *shape):
    return synth.normal(7, "llmpath." + name, shape, 1.0)


def causal(n, window=0, sinks=0):
    return torch.stack([R.visible(n, i, window, sinks) for i in range(n)])


def decoder(w, emb, sees, int4=False):
    """emb [n][1536], token i at position i, which sees the rows j with sees[i][j] -> hidden [n][1536]."""
    x = torch.from_numpy(np.ascontiguousarray(emb)).double().cuda()
    n = x.shape[0]
    hidden_rows = ~sees.cuda()
    ang = torch.arange(n).double()[:, None] * ((1e6 ** (-2.0 / 128)) ** torch.arange(64).double())[None]
    cs, sn = torch.cos(ang).cuda()[:, None], torch.sin(ang).cuda()[:, None]

    def norm(v, g):
        return v / torch.sqrt((v * v).mean(-1, keepdim=True) + 1e-6) * g

    def rope(v):
        a, b = v[..., :64], v[..., 64:]
        return torch.cat([a * cs - b * sn, b * cs + a * sn], -1)

    for l in range(LAYERS):
        p = f"llm.model.layers.{l}."
        y = norm(x, w[p + "input_layernorm.weight"])

        def lin(name):
            z = y @ w[p + f"self_attn.{name}.weight"].T
            b = w.get(p + f"self_attn.{name}.bias")
            return z if b is None else z + b

        q, k, v = rope(lin("q_proj").view(n, 12, 128)), rope(lin("k_proj").view(n, 2, 128)), lin("v_proj").view(n, 2, 128)
        k, v = (R.held(t.to(torch.bfloat16), int4) for t in (k, v))
        s = torch.einsum("ihgd,jhd->hgij", q.view(n, 2, 6, 128), k) * 128 ** -0.5
        s.masked_fill_(hidden_rows, float("-inf"))
        y = torch.einsum("hgij,jhd->ihgd", torch.softmax(s, -1), v).reshape(n, 1536)
        x = x + y @ w[p + "self_attn.o_proj.weight"].T
        if p + "self_attn.o_proj.bias" in w:
            x = x + w[p + "self_attn.o_proj.bias"]
        y = norm(x, w[p + "post_attention_layernorm.weight"])
        g = y @ w[p + "mlp.gate_proj.weight"].T
        x = x + (g / (1 + torch.exp(-g)) * (y @ w[p + "mlp.up_proj.weight"].T)) @ w[p + "mlp.down_proj.weight"].T
    return norm(x, w["llm.model.norm.weight"]).cpu().numpy()


def check(w, got, emb, sees, dtype, first, what):
    """got: the hidden rows from `first` on."""
    want = decoder(w, emb, sees, dtype == I4)[first:]
    if dtype == I4:
        # a bf16-sized difference before the rounding to 4 bits moves single codes by a step: the engine stays as close
        # to the unrounded decoder as the 64-bit decoder with 4-bit rows does
        assert_no_worse_than_recipe(got, want, decoder(w, emb, sees, False)[first:], what)
    else:
        assert_bf16_close(got, want, what)


@pytest.mark.parametrize("dtype", [BF, I4])
@pytest.mark.parametrize("window,sinks", [(0, 0), (70, 5)])
def test_prompts_of_more_than_256_tokens_and_what_follows(wide, llm, dtype, window, sinks):
    """Ragged prompts through the products of many rows, then steps, then a mixed call of many rows again."""
    lens = [200, 129, 1]
    kv = llm.kv_cache(64, 4, 16, dtype)
    seqs = [kv.open() for _ in lens]
    x = [emb_of(f"p{b}", 300, 1536) for b in range(3)]
    got = [[] for _ in lens]
    at = [0, 0, 0]
    for news in (lens, [1, 1, 1], [1, 1, 1], [40, 1, 250], [1, 1, 1]):
        rows = np.concatenate([x[b][at[b]:at[b] + n] for b, n in enumerate(news)])
        out = llm.extend(kv, seqs, news, rows, window=window, sinks=sinks)
        row = 0
        for b, n in enumerate(news):
            got[b].append(out[row:row + n])
            row += n
            at[b] += n
    for b in range(3):
        check(wide, np.concatenate(got[b]), x[b][:at[b]], causal(at[b], window, sinks), dtype, 0, f"stream {b}")
    kv.close()


@pytest.mark.parametrize("dtype", [BF, I4])
@pytest.mark.parametrize("window,sinks", [(0, 0), (900, 10)])
def test_steps_as_key_ranges_are_split_into_more_parts(wide, llm, dtype, window, sinks):
    """A stream that grows from 60 to 1500 rows beside one of 20: its steps take one part, then several, and graphs of
    other splits."""
    kv = llm.kv_cache(128, 2, 16, dtype)
    s, t = kv.open(), kv.open()
    x, y = emb_of("long", 1520, 1536), emb_of("short", 40, 1536)
    got, short = [], [llm.extend(kv, [t], [20], y[:20], window=window, sinks=sinks)]
    n, m = 0, 20
    for to in (60, 130, 300, 620, 1000, 1490):
        got.append(llm.extend(kv, [s], [to - n], x[n:to], window=window, sinks=sinks))
        n = to
        for _ in range(2):
            out = llm.extend(kv, [s, t], [1, 1], np.stack([x[n], y[m]]), window=window, sinks=sinks)
            got.append(out[:1])
            short.append(out[1:])
            n, m = n + 1, m + 1
    check(wide, np.concatenate(got), x[:n], causal(n, window, sinks), dtype, 0, "growing stream")
    check(wide, np.concatenate(short), y[:m], causal(m, window, sinks), dtype, 0, "short stream")
    kv.close()


@pytest.mark.parametrize("dtype", [BF, I4])
@pytest.mark.parametrize("window,sinks", [(0, 0), (30, 4)])
def test_a_compacted_sequence_goes_on(wide, llm, dtype, window, sinks):
    """Kept rows stay those of their old positions; new tokens take the positions behind the old length, and a window
    counts the rows that are held."""
    n, more = 100, 33
    keep = [0, 1, 2, 3] + list(range(9, 60, 3)) + list(range(80, 95))
    x = emb_of("compact", n + more, 1536)
    kv = llm.kv_cache(32, 3, 16, dtype)
    s = kv.open()
    llm.extend(kv, [s], [n], x[:n])
    (f,) = kv.fork(s)
    kv.compact(f, keep)
    assert kv.length(f) == len(keep) and kv.position(f) == n
    got = [llm.extend(kv, [f], [30], x[n:n + 30], window=window, sinks=sinks)]
    got += [llm.extend(kv, [f], [1], x[i:i + 1], window=window, sinks=sinks) for i in range(n + 30, n + more)]
    assert kv.length(f) == len(keep) + more and kv.position(f) == n + more
    sees = torch.zeros(n + more, n + more, dtype=torch.bool)
    sees[:n, :n] = causal(n)
    held = torch.tensor(keep + list(range(n, n + more)))
    rows = causal(len(held), window, sinks)
    for i in range(more):
        sees[n + i, held] = rows[len(keep) + i]
    check(wide, np.concatenate(got), x, sees, dtype, n, "compacted")
    step = llm.extend(kv, [s], [1], x[n:n + 1])            # the source knows nothing of it
    check(wide, step, x[:n + 1], causal(n + 1), dtype, n, "its source")
    kv.close()


def test_more_step_graphs_than_are_kept(wide, llm):
    """Steps with over 64 windows between dense steps: every one is right, before and after graphs are dropped."""
    kv = llm.kv_cache(64, 2, 16)
    s = kv.open()
    x = emb_of("churn", 100, 1536)
    dense = emb_of("dense", 2, 60, 1536)
    got = [llm.extend(kv, [s], [20], x[:20])]
    llm.prefill(dense[:, :4])
    steps = []
    for i in range(70):
        got.append(llm.extend(kv, [s], [1], x[20 + i:21 + i], window=5 + i % 68, sinks=1))
        if i % 2:
            steps.append(llm.step(dense[:, 4 + i // 2]))
    sees = causal(90)
    for i in range(70):
        sees[20 + i] = R.visible(90, 20 + i, 5 + i % 68, 1)
    check(wide, np.concatenate(got), x[:90], sees, BF, 0, "windows")
    for b in range(2):
        check(wide, np.stack([o[b] for o in steps]), dense[b, :39], causal(39), BF, 4, f"dense sequence {b}")
    kv.close()


def test_step_graphs_in_use_outlive_the_others(wide, weights):
    """Over 64 windows take the place of the least recently used paged graph only.  The legacy default stream (handle 1)
    runs a graph but captures none, so a step on it works where its graph is there."""
    llm = dtts.LLM(weights, n_layers=LAYERS, max_batch=2, max_seq=256)
    kv = llm.kv_cache(32, 2, 16)
    s = kv.open()
    x = emb_of("kept", 200, 1536)
    dense = emb_of("keptdense", 2, 6, 1536)
    llm.prefill(dense[:, :4])
    last = llm.step(dense[:, 4])
    got, windows = [llm.extend(kv, [s], [20], x[:20])], []
    for i in range(70):
        for w in (4, 5 + i):
            n = 20 + len(windows)
            got.append(llm.extend(kv, [s], [1], x[n:n + 1], window=w))
            windows.append(w)
    torch.cuda.synchronize()
    llm.set_stream(1)
    n = 20 + len(windows)
    last2 = llm.step(dense[:, 5])                                    # the dense step's
    got.append(llm.extend(kv, [s], [1], x[n:n + 1], window=4))       # the one of every other step
    got.append(llm.extend(kv, [s], [1], x[n + 1:n + 2], window=74))  # the newest
    with pytest.raises(dtts.DttsError):
        llm.extend(kv, [s], [1], x[n + 2:n + 3], window=5)           # the oldest
    windows += [4, 74]
    torch.cuda.synchronize()
    llm.set_stream(None)
    assert kv.length(s) == n + 2
    sees = causal(n + 2)
    for i, w in enumerate(windows):
        sees[20 + i] = R.visible(n + 2, 20 + i, w, 0)
    check(wide, np.concatenate(got), x[:n + 2], sees, BF, 0, "windows")
    for b in range(2):
        check(wide, np.stack([last[b], last2[b]]), dense[b], causal(6), BF, 4, f"dense sequence {b}")
    kv.close()
    llm.close()


def test_prompts_past_32_bit_offsets(llm):
    """64 prompts of 2000 tokens: 17920 columns of gate and up projections pass 2^31 elements.  The first and the last
    stream come out as they do alone."""
    n, rows = 64, 2000
    assert n * rows * 17920 > 2 ** 31
    g = torch.Generator(device="cuda")
    g.manual_seed(5)
    x = torch.randn(n * rows, 1536, device="cuda", generator=g)
    out = torch.empty_like(x)
    kv = llm.kv_cache(n * (rows // 64 + 1) + 40, n + 1, 64)
    seqs = [kv.open() for _ in range(n)]
    torch.cuda.synchronize()
    llm.extend(kv, seqs, [rows] * n, x, out=out, mem=dtts.MEM_DEVICE)
    kv.sync()
    for b in (0, n - 1):
        s = kv.open()
        part, alone = x[b * rows:(b + 1) * rows].cpu().numpy(), out[b * rows:(b + 1) * rows].cpu().numpy()
        assert_bf16_close(llm.extend(kv, [s], [rows], part), alone, f"stream {b}")
        kv.close_seqs([s])
    kv.close()
