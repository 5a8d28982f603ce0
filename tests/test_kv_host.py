"""Host-side checks of the paged K/V cache that need no GPU: refusals before any device is touched, and the
definition of 4-bit rows the GPU tests rely on."""
import ctypes as C

import numpy as np
import pytest
import torch

import dtts
import kv_ref as R


def _config(**change):
    c = dict(n_layers=2, n_kv_heads=2, head_dim=128, page_tokens=64, n_pages=8, max_seqs=2, max_tokens=256,
             dtype=dtts.DTYPE_INT4)
    c.update(change)
    return dtts.KVConfig(*[c[n] for n, _ in dtts.KVConfig._fields_])


@pytest.mark.parametrize("change,status", [
    (dict(dtype=dtts.DTYPE_FP8), dtts.ERR_UNSUPPORTED), (dict(dtype=dtts.DTYPE_F32), dtts.ERR_UNSUPPORTED),
    (dict(dtype=9), dtts.ERR_UNSUPPORTED), (dict(head_dim=96), dtts.ERR_UNSUPPORTED), (dict(head_dim=0), dtts.ERR_UNSUPPORTED),
    (dict(page_tokens=8), dtts.ERR_UNSUPPORTED), (dict(page_tokens=48), dtts.ERR_UNSUPPORTED),
    (dict(page_tokens=256), dtts.ERR_UNSUPPORTED), (dict(n_layers=0), dtts.ERR_ARG), (dict(n_layers=-1), dtts.ERR_ARG),
    (dict(n_kv_heads=0), dtts.ERR_ARG), (dict(n_layers=1000, n_kv_heads=100), dtts.ERR_ARG), (dict(n_pages=0), dtts.ERR_ARG),
    (dict(max_seqs=0), dtts.ERR_ARG), (dict(max_seqs=65536), dtts.ERR_ARG), (dict(max_tokens=0), dtts.ERR_ARG),
    (dict(max_tokens=(1 << 24) + 1), dtts.ERR_ARG), (dict(max_seqs=60000, max_tokens=1 << 24, page_tokens=16), dtts.ERR_ARG)])
def test_bad_configurations_are_refused(dtts_mod, change, status):
    h = C.c_void_p(5)
    assert dtts.lib().dtts_kv_create(C.byref(_config(**change)), 0, C.byref(h)) == status
    assert not h.value and dtts.lib().dtts_last_error()


def test_null_arguments_are_refused(dtts_mod):
    L = dtts.lib()
    n = C.c_int()
    h = C.c_void_p()
    assert L.dtts_kv_create(None, 0, C.byref(h)) == dtts.ERR_ARG
    assert L.dtts_kv_create(C.byref(_config()), 0, None) == dtts.ERR_ARG
    assert L.dtts_kv_destroy(None) == dtts.OK
    calls = [L.dtts_kv_set_stream(None, None), L.dtts_kv_sync(None), L.dtts_kv_open(None, C.byref(n)),
             L.dtts_kv_close(None, 0, None), L.dtts_kv_fork(None, 0, 0, None), L.dtts_kv_truncate(None, 0, 0),
             L.dtts_kv_trim(None, 0, 1, 0), L.dtts_kv_compact(None, 0, 0, None), L.dtts_kv_length(None, 0, None, None),
             L.dtts_kv_free_pages(None, C.byref(n)), L.dtts_kv_extend(None, 1, None, None),
             L.dtts_kv_write(None, 0, None, None, 0, 0, 0, 0), L.dtts_kv_attend(None, 0, None),
             L.dtts_kv_read(None, 0, 1, 0, None, None, None, None, None, dtts.DTYPE_F32),
             L.dtts_llm_kv_create(None, 1, 1, 64, dtts.DTYPE_BF16, C.byref(h)),
             L.dtts_llm_extend(None, None, 1, None, None, None, 0, 0, None, dtts.MEM_HOST)]
    assert calls == [dtts.ERR_ARG] * len(calls)


def test_no_device_is_an_error(dtts_mod):
    if dtts_mod.device_count() > 0:
        pytest.skip("a device is visible here")
    h = C.c_void_p()
    assert dtts.lib().dtts_kv_create(C.byref(_config()), 0, C.byref(h)) == dtts.ERR_NO_DEVICE and not h.value


def test_four_bit_rows_are_within_half_a_step():
    g = torch.Generator()
    g.manual_seed(1)
    x = (torch.randn(64, 3, 128, generator=g) * torch.logspace(-3, 3, 64)[:, None, None]).bfloat16()
    c, s = R.codes(x)
    assert c.abs().max() == 7 and torch.equal(s.to(torch.float16).double(), s)
    err = (R.held(x, True) - x.double()).reshape(64, 3, 4, 32).abs()
    # half a step, and where bf16(max / 7) was rounded down the largest value is clamped: 7 * 2^-8 of a step more
    assert (err <= s * (0.5 + 7 * 2.0 ** -8)).all()
    # every value is exact in half
    assert torch.equal(R.held(x, True).to(torch.float16).double(), R.held(x, True))


def test_host_tensors_and_other_types_are_refused():
    """The Python calls look at shapes, types and devices before the library sees an address."""
    kv = dtts.KVCache.__new__(dtts.KVCache)
    kv._init(None, 1, 2, 64, 0)
    kv._rows = 2
    host = torch.zeros(2, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="on device 0"):
        kv.write(0, host, host)
    with pytest.raises(ValueError, match="on device 0"):
        kv.attend(0, host, host)
    with pytest.raises(ValueError, match="on device 0"):
        kv.read(0, [0], [0], [2], torch.zeros(1, 2, 2, 64), torch.zeros(1, 2, 2, 64))
    with pytest.raises(ValueError):
        kv.extend([0, 1], [1])


def _llm_and_cache():
    kv = dtts.KVCache.__new__(dtts.KVCache)
    kv._init(None, 1, 2, 128, 0)
    e = dtts.LLM.__new__(dtts.LLM)
    e.h, e.device, e.n_layers = None, 0, 1
    return e, kv


@pytest.mark.parametrize("mem", [dtts.MEM_HOST, dtts.MEM_DEVICE])
def test_decoder_buffers_of_another_kind_are_refused(dtts_mod, mem):
    """The library writes rows x 1536 floats to out: a buffer that does not hold them is refused before the call."""
    e, kv = _llm_and_cache()
    emb = np.zeros((3, 1536), np.float32)
    frozen = np.zeros((3, 1536), np.float32)
    frozen.flags.writeable = False
    bad = [np.zeros((3, 1536), t) for t in (np.float16, np.float64, np.int8)]
    bad += [np.zeros((2, 1536), np.float32), np.zeros((1536, 3), np.float32), np.zeros((1536, 3), np.float32).T,
            np.zeros((6, 1536), np.float32)[::2], frozen, torch.zeros(3, 1536, dtype=torch.bfloat16),
            torch.zeros(1536, 3).T, torch.zeros(3, 1536, device="meta")]
    for out in bad:
        with pytest.raises(ValueError, match="out|emb"):
            e.extend(kv, [0], [3], emb, out=out, mem=mem)
    if mem == dtts.MEM_DEVICE:          # host memory in place of the device's
        for x in (emb, torch.zeros(3, 1536)):
            with pytest.raises(ValueError, match="on device 0"):
                e.extend(kv, [0], [3], x, out=x, mem=mem)
    else:
        for out in (None, np.zeros((3, 1536), np.float32), torch.zeros(3, 1536)):
            with pytest.raises(dtts.DttsError):        # as far as the library, which has no engine here
                e.extend(kv, [0], [3], emb, out=out, mem=mem)
        with pytest.raises(dtts.DttsError):            # emb is only read
            e.extend(kv, [0], [3], frozen, mem=mem)


@pytest.mark.parametrize("bad", [np.array([0.5]), np.array([2 ** 32 + 1]), np.array([-2 ** 31 - 1]), np.array([True]),
                                 np.array([2 ** 63], np.uint64), np.array(["1"]), range(2 ** 31, 2 ** 31 + 1)])
def test_numbers_that_are_not_32_bit_integers_are_refused(dtts_mod, bad):
    """None of them becomes another sequence or count on the way."""
    kv = dtts.KVCache.__new__(dtts.KVCache)
    kv._init(None, 1, 2, 64, 0)
    for call in (lambda: kv.extend(bad, [1]), lambda: kv.extend([1], bad), lambda: kv.close_seqs(bad), lambda: kv.compact(0, bad)):
        with pytest.raises(ValueError):
            call()
    for good in (np.array([1]), np.array([1], np.uint8), range(1, 2), torch.tensor([1])):
        assert dtts._ints(good)[0].tolist() == [1] and dtts._ints(good)[2] == 1
