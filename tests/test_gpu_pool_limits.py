"""Sessions at the end of their room on a B200: decode loops and calls that meet max_ctx or the
last page of a pool. Frames and ids are compared for equality with sessions that have room."""
import numpy as np
import pytest

import syrinx_b200 as sx
from syrinx_b200.configs import QWEN3_4B, SX_DTYPE_BF16, SX_DTYPE_F32, SX_DTYPE_Q8_0, TINY_S2, shrink
from syrinx_b200.workloads import prompt_for

pytestmark = pytest.mark.gpu
PAGE = 64


@pytest.fixture(scope="module")
def tiny():
    m = sx.Model(TINY_S2, sx.synth_blob(TINY_S2, SX_DTYPE_Q8_0, seed=7), device=0)
    yield m
    m.close()


def prompts(lengths):
    return [prompt_for(TINY_S2, T, seed=60 + T) for T in lengths]


def roomy(m, ps, frames):
    a = sx.B200DualAr(m, max_ctx=512, max_batch=len(ps))
    a.prefill_batch(ps)
    want = a.decode_greedy_batch(len(ps), frames, mask_stop=True)
    a.close()
    assert all(len(w) == frames for w in want)
    return want


@pytest.mark.parametrize("how,room", [(dict(max_ctx=512, pool_pages=4), 22), (dict(max_ctx=110), 10),
                                      (dict(max_ctx=110, pool_pages=8), 10)])
def test_batched_loop_that_ends_early_keeps_sequences_apart(tiny, how, room):
    """Three sequences ask for 30 frames where there is room for fewer: each one's frames stand in its
    own rows. Four pages hold 100 + f, 5 + f and 42 + f positions up to f = 22."""
    ps = prompts([100, 5, 42])
    want = roomy(tiny, ps, 30)
    b = sx.B200DualAr(tiny, max_batch=3, **how)
    b.prefill_batch(ps)
    got = b.decode_greedy_batch(3, 30, mask_stop=True)
    b.close()
    for g, w in zip(got, want):
        assert len(g) == room and np.array_equal(g, w[:room])


def test_batched_prefill_and_drive_report_a_failed_reset(tiny):
    """A reset that fails (its copies are refused on a stream that is being captured) ends the call with
    its own code; before, the call went on with the lengths and pages of the sequences it was to drop."""
    import ctypes as C

    torch = pytest.importorskip("torch")
    cu = C.CDLL("libcuda.so.1")
    be = sx.B200DualAr(tiny, max_ctx=128, max_batch=2, pool_pages=4)
    stream = torch.cuda.Stream()
    be.set_stream(stream.cuda_stream)
    p = prompts([100, 60])
    first = be.prefill(p[0]).semantic_logits
    torch.cuda.synchronize()
    for call in (lambda: be.prefill_batch([p[1]]), lambda: drive_c(be, p[1], 3)):
        graph = C.c_void_p()
        assert cu.cuStreamBeginCapture_v2(C.c_void_p(stream.cuda_stream), 2) == 0
        try:
            with pytest.raises(sx.SyrinxError) as e:
                call()
        finally:
            cu.cuStreamEndCapture(C.c_void_p(stream.cuda_stream), C.byref(graph))
        assert e.value.code == -2 and be.seq_len(0) == 100
    be.reset()
    assert be.pool_free() == 4 and np.array_equal(be.prefill(p[0]).semantic_logits, first)
    be.set_stream(None)
    be.close()


def drive_c(be, prompt, n):
    """sx_drive with the greedy sampler: [codebooks, frames]."""
    import ctypes as C

    from syrinx_b200 import _lib

    p = np.ascontiguousarray(prompt, dtype=np.uint32)
    out, got, params = np.zeros((be.cfg.num_codebooks, max(1, n)), np.uint32), C.c_int32(-1), sx.GREEDY.to_c()
    _lib.check(_lib.lib().sx_drive(be.handle, p.ctypes.data_as(C.POINTER(C.c_uint32)), p.shape[-1], n, 0, C.byref(params),
                                   out.ctypes.data_as(C.POINTER(C.c_uint32)), C.byref(got)))
    return out[:, : got.value]


def test_prompts_that_do_not_fit_change_nothing(tiny):
    """A batched prefill or a drive whose prompts need more pages than the pool has is refused before the
    sequences that are there are dropped: lengths and free pages stay, and decoding goes on as if it had
    not been called."""
    a = sx.B200DualAr(tiny, max_ctx=512, max_batch=2)
    b = sx.B200DualAr(tiny, max_ctx=512, max_batch=2, pool_pages=4)
    ps = prompts([100, 20])
    a.prefill_batch(ps), b.prefill_batch(ps)
    fa, fb = a.decode_greedy_batch(2, 5, mask_stop=True), b.decode_greedy_batch(2, 5, mask_stop=True)
    for call in (lambda: b.prefill_batch(prompts([100, 130])), lambda: b.prefill_batch(prompts([257])),
                 lambda: drive_c(b, prompts([257])[0], 3)):
        with pytest.raises(sx.SyrinxError) as e:
            call()
        assert e.value.code == -7 and [b.seq_len(i) for i in range(2)] == [105, 25] and b.pool_free() == 1
    fa, fb = a.decode_greedy_batch(2, 7, mask_stop=True), b.decode_greedy_batch(2, 7, mask_stop=True)
    assert all(np.array_equal(x, y) and len(y) == 7 for x, y in zip(fa, fb))
    # what fits exactly is taken
    b.prefill_batch(prompts([128, 127]))
    assert b.pool_free() == 0
    a.close()
    b.close()


@pytest.mark.parametrize("T,n_pages,room", [(100, 2, 29), (64, 1, 1), (120, 3, 40), (1, 1, 40)])
def test_drive_ends_with_the_pool(tiny, T, n_pages, room):
    """A drive that meets the last page returns the frames up to there, as at max_ctx: T + f positions
    after f steps, and a frame more, whose step is not taken."""
    p = prompts([T])[0]
    a = sx.B200DualAr(tiny, max_ctx=512)
    b = sx.B200DualAr(tiny, max_ctx=512, pool_pages=n_pages)
    want = drive_c(a, p, 40)
    ended = min(room, want.shape[1])  # a stop id may end both earlier
    assert ended >= 1
    for got in (drive_c(b, p, 40), sx.drive(b, p, 40, seed=0, sampling=sx.GREEDY)):
        assert got.shape[1] == ended and np.array_equal(got, want[:, :ended])
    a.close()
    b.close()


@pytest.mark.parametrize("kv", [SX_DTYPE_F32, SX_DTYPE_BF16])
def test_hidden_states_at_the_4b_shape(kv):
    """Four layers of the 4B shape (32 / 8 heads of 128) behind a context of 3000: a pooled session against
    a static one that is fed the same frames (codes whose logits nearly tie may fall either way).

    Bound. An attention over n positions in another order is off by at most 8 sqrt(n) u = 2.6e-5 of its
    size, and four layers that pass it on at twice its relative size come to 4e-4 of the hidden state's.
    A bf16 cache may round a new key the other way, 2^-8 of an element: with |q k| up to 10 and a scale of
    1 / sqrt(128), a score by 3.5e-3 and, were all the weight on it, the result by as much: 4e-3."""
    cfg = shrink(QWEN3_4B, 4, 2)
    m = sx.Model(cfg, sx.synth_blob(cfg, SX_DTYPE_Q8_0, seed=3), device=0)
    a = sx.B200DualAr(m, max_ctx=4096, kv_dtype=kv)
    b = sx.B200DualAr(m, max_ctx=4096, kv_dtype=kv, pool_pages=50)
    prompt = prompt_for(cfg, 40, seed=5)
    tol = 4e-4 if kv == SX_DTYPE_F32 else 4e-3
    for be in (a, b):
        be.fill_kv_synthetic(3000, seed=4)
    x, y = a.prefill(prompt), b.prefill(prompt)
    for k in range(60):
        for p, q in ((x.hidden, y.hidden), (x.semantic_logits, y.semantic_logits)):
            assert np.max(np.abs(p - q)) <= tol * np.max(np.abs(p))
        frame, _ = a.frame_step_greedy(None, mask_stop=True)
        x, y = a.slow_step(frame, 3040 + k), b.slow_step(frame, 3040 + k)
    assert b.pool_free() == 50 - 49
    a.close()
    b.close()
    m.close()
