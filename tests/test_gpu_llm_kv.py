"""The LLM decoder over a paged cache (dtts_llm_extend) against a decoder in 64 bits over the definitions of
kv_ref, and against the reference's own src/llm_manual.cpp where its semantics apply (bf16, no window)."""
import numpy as np
import pytest
import torch

import dtts
import kv_ref as R
import synth
from helpers import assert_bf16_close, assert_no_worse_than_recipe

pytestmark = pytest.mark.gpu

LAYERS = 2


@pytest.fixture(scope="module")
def weights():
    return synth.llm_weights(3, n_layers=LAYERS)


@pytest.fixture(scope="module")
def llm(weights):
    e = dtts.LLM(weights, n_layers=LAYERS, max_batch=1, max_seq=512)
    yield e
    e.close()


def decoder(weights, emb, int4=False, window=0, sinks=0):
    """emb [n][1536] -> hidden [n][1536] in 64 bits, K/V rounded as the cache holds them."""
    w = {k: torch.from_numpy(np.ascontiguousarray(v)).double() for k, v in weights.items() if k.startswith("llm.model.")}
    x = torch.from_numpy(np.ascontiguousarray(emb)).double()
    n = x.shape[0]
    theta = 1e6 ** (-2.0 / 128)
    ang = torch.arange(n).double()[:, None] * (theta ** torch.arange(64).double())[None]
    cs, sn = torch.cos(ang)[:, None], torch.sin(ang)[:, None]

    def norm(v, g):
        return v / torch.sqrt((v * v).mean(-1, keepdim=True) + 1e-6) * g

    def rope(v):
        a, b = v[..., :64], v[..., 64:]
        return torch.cat([a * cs - b * sn, b * cs + a * sn], -1)

    for l in range(LAYERS):
        p = f"llm.model.layers.{l}."
        y = norm(x, w[p + "input_layernorm.weight"])
        lin = lambda name: y @ w[p + f"self_attn.{name}.weight"].T + w.get(p + f"self_attn.{name}.bias", torch.zeros(1).double())
        q, k, v = (rope(lin("q_proj").view(n, 12, 128)), rope(lin("k_proj").view(n, 2, 128)), lin("v_proj").view(n, 2, 128))
        k, v = (R.held(t.to(torch.bfloat16), int4) for t in (k, v))
        o = torch.zeros(n, 12, 128).double()
        for i in range(n):
            j = R.visible(n, i, window, sinks).nonzero()[:, 0]
            s = torch.einsum("hgd,jhd->hgj", q[i].view(2, 6, 128), k[j]) * 128 ** -0.5
            o[i] = torch.einsum("hgj,jhd->hgd", torch.softmax(s, -1), v[j]).reshape(12, 128)
        x = x + o.reshape(n, 1536) @ w[p + "self_attn.o_proj.weight"].T + w.get(p + "self_attn.o_proj.bias", torch.zeros(1).double())
        y = norm(x, w[p + "post_attention_layernorm.weight"])
        g = y @ w[p + "mlp.gate_proj.weight"].T
        x = x + (g / (1 + torch.exp(-g)) * (y @ w[p + "mlp.up_proj.weight"].T)) @ w[p + "mlp.down_proj.weight"].T
    return norm(x, w["llm.model.norm.weight"]).numpy()


def emb_of(name, *shape):
    return synth.normal(5, "llmkv." + name, shape, 1.0)


def test_ragged_prompts_and_steps_match_the_reference(weights, llm, ref):
    lens, steps = [13, 40, 1], 3
    prompts = [emb_of(f"p{b}", n, 1536) for b, n in enumerate(lens)]
    step = emb_of("s", steps, 3, 1536)
    kv = llm.kv_cache(32, 4, 16)
    seqs = [kv.open() for _ in lens]
    hid = llm.extend(kv, seqs, lens, np.concatenate(prompts))
    outs = [llm.extend(kv, seqs, [1, 1, 1], step[i]) for i in range(steps)]
    assert [kv.length(s) for s in seqs] == [n + steps for n in lens]
    at = 0
    for b, n in enumerate(lens):
        want_p, want_s = ref.llm_run(weights, LAYERS, prompts[b], step[:, b])
        assert_bf16_close(hid[at:at + n], want_p, f"prompt {b}")
        assert_bf16_close(np.stack([o[b] for o in outs]), want_s, f"steps {b}")
        at += n
    kv.close()


@pytest.mark.parametrize("window,sinks", [(0, 0), (16, 3)])
@pytest.mark.parametrize("dtype", [dtts.DTYPE_BF16, dtts.DTYPE_INT4])
def test_streams_fork_continue_and_end(weights, llm, dtype, window, sinks):
    """A voice prompt, two continuations from it, a third stream joining in mixed batches, trimmed pages."""
    int4 = dtype == dtts.DTYPE_INT4
    base, a, b, c = emb_of("base", 37, 1536), emb_of("a", 9, 1536), emb_of("b", 9, 1536), emb_of("c", 25, 1536)
    kv = llm.kv_cache(24, 4, 16, dtype)
    s0 = kv.open()
    got = {s0: [llm.extend(kv, [s0], [37], base, window=window, sinks=sinks)]}
    (s1,) = kv.fork(s0)
    s2 = kv.open()
    got[s1], got[s2] = [], []
    feed = {s0: a, s1: b, s2: c}
    used = {s: 0 for s in feed}
    for news in ([1, 1, 20], [1, 1, 1], [3, 1, 1], [0, 2, 1], [1, 1, 0]):
        rows = []
        for s, n in zip((s0, s1, s2), news):
            rows.append(feed[s][used[s]:used[s] + n])
            used[s] += n
        if window:
            for s in (s0, s1, s2):
                kv.trim(s, window, sinks)
        out = llm.extend(kv, [s0, s1, s2], news, np.concatenate(rows), window=window, sinks=sinks)
        at = 0
        for s, n in zip((s0, s1, s2), news):
            got[s].append(out[at:at + n])
            at += n
    for s, e, skip in ((s0, np.concatenate([base, a]), 0), (s1, np.concatenate([base, b]), 37), (s2, c, 0)):
        g = np.concatenate(got[s])
        e = e[:skip + len(g)]
        want = decoder(weights, e, int4, window, sinks)[skip:]
        if int4:
            # a bf16-sized difference before the rounding to 4 bits moves single codes by a step: the engine stays
            # as close to the unrounded decoder as the 64-bit decoder with 4-bit rows does
            assert_no_worse_than_recipe(g, want, decoder(weights, e, False, window, sinks)[skip:], f"stream {s}")
        else:
            assert_bf16_close(g, want, f"stream {s}")
    free = kv.free_pages()
    kv.close_seqs([s0, s1, s2])
    assert kv.free_pages() == 24 > free
    kv.close()


def test_steps_keep_one_graph_as_streams_grow(weights, llm):
    """Captured steps read lengths and tables on the device: a stream that grows over pages and beside one
    that is replaced in mid-flight."""
    kv = llm.kv_cache(64, 4, 16)
    e = emb_of("grow", 120, 1536)
    f = emb_of("other", 120, 1536)
    s, t = kv.open(), kv.open()
    got = [llm.extend(kv, [s, t], [1, 1], np.stack([e[i], f[i]])) for i in range(60)]
    kv.close_seqs([t])
    t2 = kv.open()
    got2 = [llm.extend(kv, [s, t2], [1, 1], np.stack([e[60 + i], f[i]])) for i in range(60)]
    want, want_f = decoder(weights, e), decoder(weights, f[:60])
    assert_bf16_close(np.stack([g[0] for g in got + got2]), want, "growing stream")
    assert_bf16_close(np.stack([g[1] for g in got]), want_f, "second stream")
    assert_bf16_close(np.stack([g[1] for g in got2]), want_f, "its successor")
    kv.close()


def test_refusals_change_nothing(llm):
    kv = llm.kv_cache(4, 2, 16)
    s = kv.open()
    x = emb_of("r", 65, 1536)
    with pytest.raises(dtts.DttsError) as e:
        llm.extend(kv, [s], [65], x)                      # 5 pages of 4
    assert e.value.status == dtts.ERR_OOM and kv.length(s) == 0 and kv.free_pages() == 4
    with pytest.raises(dtts.DttsError):
        llm.extend(kv, [s, s], [1, 1], x[:2])
    with pytest.raises(dtts.DttsError):
        llm.extend(kv, [1], [1], x[:1])
    with pytest.raises(dtts.DttsError):
        llm.extend(kv, [s], [1], x[:1], window=-1)
    with pytest.raises(dtts.DttsError):
        llm.extend(kv, [s], [513], emb_of("long", 513, 1536))   # beyond max_seq
    other = dtts.KVCache(LAYERS + 1, 2, 128, 4, 1, 64)
    o = other.open()
    with pytest.raises(dtts.DttsError):
        llm.extend(other, [o], [1], x[:1])
    other.close()
    assert kv.length(s) == 0 and kv.free_pages() == 4
    llm.extend(kv, [s], [0], x[:0])
    llm.extend(kv, [s], [40], x[:40])
    kv.trim(s, 4)
    with pytest.raises(dtts.DttsError):
        llm.extend(kv, [s], [1], x[:1])                   # the whole history, parts of which are freed
    assert kv.length(s) == 40
    assert np.isfinite(llm.extend(kv, [s], [1], x[:1], window=4)).all()
    kv.close()


def test_capturing_streams_are_refused(weights):
    """A call while the cache's stream or the engine's is capturing changes nothing."""
    e = dtts.LLM(weights, n_layers=LAYERS, max_batch=1, max_seq=64)
    kv = e.kv_cache(8, 2, 16)
    s = kv.open()
    x = emb_of("capture", 4, 1536)
    e.extend(kv, [s], [2], x[:2])
    st = torch.cuda.Stream()
    y = torch.zeros(8, device="cuda")
    for mine in (kv, e):
        mine.set_stream(st.cuda_stream)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.stream(st):
            with torch.cuda.graph(graph, stream=st, capture_error_mode="thread_local"):
                y.add_(1)
                with pytest.raises(dtts.DttsError) as err:
                    e.extend(kv, [s], [1], x[2:3])
        assert err.value.status == dtts.ERR_UNSUPPORTED and kv.length(s) == 2
        graph.replay()
        torch.cuda.synchronize()
        mine.set_stream(None)
    want = decoder(weights, x)
    assert_bf16_close(e.extend(kv, [s], [2], x[2:]), want[2:], "after the refusals")
    kv.close()
    e.close()


@pytest.mark.parametrize("dense", [False, True])
def test_a_workspace_that_does_not_fit_leaves_the_engine_usable(weights, dense):
    """1.7 million tokens need 198 GB of workspace (116224 bytes each), more than the device has, beside pages for
    all of them; the next calls, above and below 256 tokens, work on a workspace of their own."""
    n, rows = 416, 4096
    e = dtts.LLM(weights, n_layers=LAYERS, max_batch=n if dense else 1, max_seq=rows)
    kv = e.kv_cache(n * rows // 128, n, 128)
    x = emb_of("fit", 303, 1536)
    s = kv.open()
    e.extend(kv, [s], [2], x[:2])                          # a small workspace is there before
    seqs = [s] + [kv.open() for _ in range(n - 1)]
    free, small = kv.free_pages(), torch.zeros(16, device="cuda")
    counts = [rows - 2] + [rows] * (n - 1)
    ps, pc = dtts._ints(seqs), dtts._ints(counts)
    if dense:
        st = dtts.lib().dtts_llm_prefill(e.h, small.data_ptr(), n, rows, small.data_ptr(), dtts.MEM_DEVICE)
    else:
        st = dtts.lib().dtts_llm_extend(e.h, kv.h, n, ps[1], pc[1], small.data_ptr(), 0, 0, small.data_ptr(), dtts.MEM_DEVICE)
    assert st == dtts.ERR_OOM
    assert [kv.length(q) for q in seqs] == [2] + [0] * (n - 1) and kv.free_pages() == free
    want = decoder(weights, x)
    assert_bf16_close(e.extend(kv, [s], [1], x[2:3]), want[2:3], "a step")
    assert_bf16_close(e.extend(kv, [s], [299], x[3:302]), want[3:302], "a prompt")
    assert_bf16_close(e.extend(kv, [s], [1], x[302:]), want[302:], "the next step")
    kv.close()
    e.close()


def test_an_error_behind_the_growth_takes_it_back(weights):
    """A step on the legacy default stream fails where it would be captured: lengths, positions, pages (a fork's shared
    one among them) and the rows are as they were, and the batch is over."""
    e = dtts.LLM(weights, n_layers=LAYERS, max_batch=1, max_seq=128)
    kv = e.kv_cache(12, 4, 16)
    x, y = emb_of("back", 45, 1536), emb_of("back2", 45, 1536)
    a, b = kv.open(), kv.open()
    e.extend(kv, [a, b], [40, 16], np.concatenate([x[:40], y[:16]]))
    (f,) = kv.fork(a)
    free = kv.free_pages()
    assert free == 12 - 4
    for _ in range(2):
        torch.cuda.synchronize()
        e.set_stream(1)
        with pytest.raises(dtts.DttsError) as err:
            e.extend(kv, [f, b, a], [1, 1, 1], np.stack([x[40], y[16], x[40]]))
        torch.cuda.synchronize()
        e.set_stream(None)
        assert err.value.status == dtts.ERR_CUDA
        assert [kv.length(s) for s in (a, b, f)] == [kv.position(s) for s in (a, b, f)] == [40, 16, 40]
        assert kv.free_pages() == free
        with pytest.raises(dtts.DttsError):        # no batch is current
            kv.write(0, torch.zeros(3, 2, 128, dtype=torch.bfloat16, device="cuda"),
                     torch.zeros(3, 2, 128, dtype=torch.bfloat16, device="cuda"))
    out = [e.extend(kv, [f, b, a], [1, 1, 1], np.stack([y[i - 24], y[i - 24], x[i]])) for i in (40, 41, 42)]
    assert_bf16_close(np.stack([o[2] for o in out]), decoder(weights, x[:43])[40:], "the source")
    assert_bf16_close(np.stack([o[1] for o in out]), decoder(weights, y[:19])[16:], "the other stream")
    assert_bf16_close(np.stack([o[0] for o in out]), decoder(weights, np.concatenate([x[:40], y[16:19]]))[40:], "the fork")
    kv.close_seqs([a, b, f])
    assert kv.free_pages() == 12
    kv.close()
    e.close()
