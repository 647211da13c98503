"""Refusals of the decoding operators that need no GPU: every bad argument is an error before any device work."""
import ctypes

import pytest

torch = pytest.importorskip("torch")

from nspeech_b200 import lib as L  # noqa: E402


@pytest.fixture(scope="module")
def lib():
    return L.load()


BUF = ctypes.create_string_buffer(4096)
PTR = (ctypes.addressof(BUF) + 255) // 256 * 256  # an aligned address that no call may touch


def rows(ptr=PTR, ts=64, hs=64):
    return L.Rows(ptr, ts, hs)


def attend(lib, q=None, dtype=L.NQ_BF16, seqs=1, nq=4, nk=4, hq=2, hk=1, d=64, sinks=0, q_off=None, k_off=None, k=None):
    r = [q or rows(), k or rows(), rows(), rows()]
    return lib.nq_window_attention(*(ctypes.byref(x) for x in r), dtype, seqs, nq, nk, q_off, k_off, None, None, hq, hk, d, -1, 0,
                                   sinks, 0.1, None, 0, None)


@pytest.mark.parametrize("change,code", [
    (dict(dtype=7), L.NQ_ERR_DTYPE), (dict(seqs=-1), L.NQ_ERR_ARG), (dict(nq=-1), L.NQ_ERR_ARG), (dict(sinks=-1), L.NQ_ERR_ARG),
    (dict(hq=3, hk=2), L.NQ_ERR_SHAPE), (dict(hk=0), L.NQ_ERR_SHAPE), (dict(d=0), L.NQ_ERR_SHAPE), (dict(d=129), L.NQ_ERR_SHAPE),
    (dict(seqs=3), L.NQ_ERR_SHAPE), (dict(seqs=2, nk=5), L.NQ_ERR_SHAPE), (dict(nq=1 << 31), L.NQ_ERR_SHAPE),
    (dict(nk=1 << 31), L.NQ_ERR_SHAPE), (dict(q=rows(None)), L.NQ_ERR_ARG), (dict(k=rows(None)), L.NQ_ERR_ARG),
    (dict(q=rows(PTR + 1)), L.NQ_ERR_ALIGN), (dict(q=rows(ts=-1)), L.NQ_ERR_SHAPE)])
def test_window_attention_refuses(lib, change, code):
    assert attend(lib, **change) == code
    assert L.last_error()


def test_window_attention_without_work(lib):
    assert attend(lib, seqs=0) == L.NQ_OK
    assert attend(lib, nq=0) == L.NQ_OK
    assert lib.nq_window_attention(None, None, None, None, 1, 1, 1, 1, None, None, None, None, 1, 1, 64, -1, 0, 0, 1.0, None, 0,
                                   None) == L.NQ_ERR_ARG
    assert lib.nq_window_attention_workspace(L.NQ_BF16, 1, 1, 100000, 8, 8, 64, -1, 0, 0) > 0
    assert lib.nq_window_attention_workspace(L.NQ_BF16, 1, 100000, 100000, 8, 8, 64, -1, 0, 0) == 0  # rows enough
    assert lib.nq_window_attention_workspace(L.NQ_BF16, 1, 1, 1, 8, 3, 64, -1, 0, 0) == L.NQ_ERR_SHAPE


def cache(**change):
    c = dict(k=PTR, v=PTR, table=PTR, lens=PTR, refs=PTR, state=PTR, dtype=L.NQ_BF16, layers=2, pages=10, page_tokens=16,
             kv_heads=2, head_dim=64, slots=4, max_pages=5)
    c.update(change)
    return L.Cache(*(c[n] for n, _ in L.Cache._fields_))


BAD_CACHES = [(dict(k=None), L.NQ_ERR_ARG), (dict(state=None), L.NQ_ERR_ARG), (dict(dtype=2), L.NQ_ERR_DTYPE),
              (dict(page_tokens=12), L.NQ_ERR_SHAPE), (dict(page_tokens=4), L.NQ_ERR_SHAPE), (dict(page_tokens=2048), L.NQ_ERR_SHAPE),
              (dict(layers=0), L.NQ_ERR_SHAPE), (dict(head_dim=130), L.NQ_ERR_SHAPE), (dict(pages=0), L.NQ_ERR_SHAPE),
              (dict(pages=(1 << 20) + 1), L.NQ_ERR_SHAPE), (dict(slots=0), L.NQ_ERR_SHAPE), (dict(max_pages=1 << 27), L.NQ_ERR_SHAPE),
              (dict(page_tokens=1024, kv_heads=4096, head_dim=128, dtype=L.NQ_F32), L.NQ_ERR_SHAPE),
              (dict(v=PTR + 8), L.NQ_ERR_ALIGN)]


@pytest.mark.parametrize("change,code", BAD_CACHES)
def test_cache_calls_refuse_a_bad_cache(lib, change, code):
    p, r = ctypes.byref(cache(**change)), ctypes.byref(rows())
    assert lib.nq_cache_reserve(p, 0, 1, None, 1, None) == code
    assert lib.nq_cache_write(p, r, r, 0, 0, 0, 1, 1, 0, 1, None, 1, None) == code
    assert lib.nq_cache_attention(p, 0, r, r, 0, 1, 1, None, 2, -1, 0, 0, 1.0, None, 0, None) == code
    assert lib.nq_cache_fork(p, 0, 1, None, None) == code
    assert lib.nq_cache_trim(p, 0, 1, 0, 1, None) == code
    assert lib.nq_cache_compact(p, None) == code
    assert lib.nq_cache_status(p, None, None) == code


def test_cache_calls_refuse_bad_arguments(lib):
    p, r = ctypes.byref(cache()), ctypes.byref(rows())
    for first, n in ((-1, 1), (0, 5), (4, 1), (0, -1)):
        assert lib.nq_cache_reserve(p, first, n, None, 1, None) == L.NQ_ERR_SHAPE
        assert lib.nq_cache_fork(p, first, n, None, None) == L.NQ_ERR_SHAPE
        assert lib.nq_cache_trim(p, first, n, 0, 1, None) == L.NQ_ERR_SHAPE
        assert lib.nq_cache_attention(p, 0, r, r, first, n, 4, PTR, 2, -1, 0, 0, 1.0, None, 0, None) == L.NQ_ERR_SHAPE
    assert lib.nq_cache_reserve(p, 0, 1, None, -1, None) == L.NQ_ERR_ARG
    assert lib.nq_cache_trim(p, 0, 1, -1, 0, None) == L.NQ_ERR_ARG
    assert lib.nq_cache_write(p, r, r, 0, 0, 1, 2, 1, 0, 1, None, 1, None) == L.NQ_ERR_SHAPE  # layers [1, 3) of 2
    assert lib.nq_cache_write(p, r, r, 0, 0, 0, 1, 3, 0, 2, None, 1, None) == L.NQ_ERR_SHAPE  # 3 rows for 2 slots of 1
    assert lib.nq_cache_attention(p, 2, r, r, 0, 1, 1, None, 2, -1, 0, 0, 1.0, None, 0, None) == L.NQ_ERR_SHAPE
    assert lib.nq_cache_attention(p, 0, r, r, 0, 1, 1, None, 3, -1, 0, 0, 1.0, None, 0, None) == L.NQ_ERR_SHAPE
    many = ctypes.byref(cache(slots=5000))
    assert lib.nq_cache_reserve(many, 0, 4097, None, 1, None) == L.NQ_ERR_SHAPE
    assert lib.nq_cache_state_ints(0, 1) == L.NQ_ERR_SHAPE


def test_beam_calls_refuse(lib):
    def select(items=1, beams=2, vocab=10, ld=10, dtype=L.NQ_F32):
        return lib.nq_beam_select(PTR, dtype, ld, items, beams, vocab, PTR, None, 0, PTR, PTR, PTR, None, PTR, 1 << 20, None)

    assert select(dtype=3) == L.NQ_ERR_DTYPE
    for change in (dict(beams=0), dict(beams=33), dict(items=-1), dict(vocab=0), dict(ld=9), dict(items=40000)):
        assert select(**change) == L.NQ_ERR_SHAPE, change
    one = (ctypes.c_void_p * 1)(PTR)
    size = (ctypes.c_int64 * 1)(16)
    assert lib.nq_beam_reorder(one, one, size, size, size, 17, 2, PTR, None) == L.NQ_ERR_SHAPE
    assert lib.nq_beam_reorder(one, one, size, size, size, 1, 12289, PTR, None) == L.NQ_ERR_SHAPE


def test_beam_reorder_refuses_outputs_that_overlap(lib):
    def reorder(src, dst, row=16, src_by=64, dst_by=64):
        n = len(src)
        ints = [(ctypes.c_int64 * n)(*([x] * n)) for x in (row, src_by, dst_by)]
        return lib.nq_beam_reorder((ctypes.c_void_p * n)(*src), (ctypes.c_void_p * n)(*dst), *ints, n, 4, PTR, None)

    for src, dst in (([PTR, PTR], [PTR, PTR]),                          # one state twice, in place
                     ([PTR, PTR + 256], [PTR + 512, PTR + 512]),        # one output twice
                     ([PTR, PTR + 256], [PTR + 256, PTR + 512]),        # an output that is another's state
                     ([PTR], [PTR + 64]),                               # the state's second row on
                     ([PTR, PTR + 16], [PTR + 512, PTR + 520])):        # rows that meet halfway
        assert reorder(src, dst) == L.NQ_ERR_ARG, (src, dst)
        assert "overlap" in L.last_error()
    assert reorder([PTR], [PTR], dst_by=32) == L.NQ_ERR_ARG             # in place, other strides
    if not torch.cuda.is_available():  # columns of one tensor, in place: the call gets as far as the device
        columns = [PTR, PTR + 16, PTR + 48]
        assert reorder(columns, columns) in (L.NQ_ERR_CUDA, L.NQ_ERR_NOT_INIT)


def test_python_refuses_host_tensors_and_misfits():
    from nspeech_b200.attention import window_attention
    from nspeech_b200.beam import beam_select
    from nspeech_b200.cache import PagedCache
    from nspeech_b200.fast_matmul import MatMulError
    t = torch.zeros((4, 2, 64))
    with pytest.raises(MatMulError, match="CUDA"):
        window_attention(t, t, t)
    with pytest.raises(MatMulError, match="fit"):
        window_attention(t, t[:, :, :32], t[:, :, :32])
    with pytest.raises(MatMulError, match="fit"):
        window_attention(t, torch.zeros((4, 3, 64)), torch.zeros((4, 3, 64)))
    with pytest.raises(MatMulError, match="dtype"):
        window_attention(t.half(), t.half(), t.half())
    with pytest.raises(MatMulError, match="heads"):
        window_attention(t[0], t[0], t[0])
    with pytest.raises(MatMulError, match="vocab"):
        beam_select(t[0], t[0])
    with pytest.raises(MatMulError, match="unit stride"):
        beam_select(t.transpose(1, 2), t[0])
    with pytest.raises(MatMulError, match="layers"):
        PagedCache(t, t, t, t, t)
