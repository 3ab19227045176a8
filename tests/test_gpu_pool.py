"""Pooled sessions (sx_session_create_pool) on a B200: the slow AR over one pool of pages, its
appends and decode attention the paged operators, against static sessions and the CPU oracle.

Frames and ids are compared for equality. Logits pass through the same products with the
attention's sums split elsewhere: the parity contract's bound of 2e-2 holds them, and they are
within 1e-3 of a static session's (f32 sums of a few thousand terms of order one, two layers)."""
import numpy as np
import pytest

import syrinx_b200 as sx
from syrinx_b200.configs import COSYVOICE2_LM, SX_DTYPE_BF16, SX_DTYPE_F32, SX_DTYPE_Q8_0, TINY_S2, shrink
from syrinx_b200.workloads import prompt_for
from oracle import oracle as oc

pytestmark = pytest.mark.gpu
PAGE = 64


@pytest.fixture(scope="module")
def tiny():
    blob = sx.synth_blob(TINY_S2, SX_DTYPE_Q8_0, seed=7)
    m = sx.Model(TINY_S2, blob, device=0)
    yield m, oc.OracleModel(TINY_S2, blob)
    m.close()


def pages(n):
    return -(-n // PAGE)


@pytest.mark.parametrize("T,frames", [(1, 3), (12, 60), (63, 5), (64, 70), (130, 20)])
def test_greedy_frames_equal_the_oracle(tiny, T, frames):
    m, om = tiny
    be = sx.B200DualAr(m, max_ctx=512, pool_pages=pages(T + frames))
    prompt = prompt_for(TINY_S2, T, seed=T)
    step = be.prefill(prompt)
    o = oc.OracleSession(om, 512, kv_bf16=False)
    ologits, _ = o.prefill(prompt)
    assert np.max(np.abs(step.semantic_logits - ologits)) <= 1e-3
    got = be.decode_greedy(frames, mask_stop=True)
    o.reset()
    want, _ = o.drive_greedy(prompt, frames, mask_stop=True)
    assert np.array_equal(got, want)
    assert be.pool_free() == 0
    be.close()


@pytest.mark.parametrize("kv", [SX_DTYPE_F32, SX_DTYPE_BF16])
def test_equals_a_static_session_call_by_call(tiny, kv):
    m, _ = tiny
    prompt = prompt_for(TINY_S2, 70, seed=3)
    outs = []
    for pool in (0, 4):
        be = sx.B200DualAr(m, max_ctx=256, kv_dtype=kv, pool_pages=pool)
        rows, frame = [be.prefill(prompt)], None
        frame, _ = be.frame_step_greedy(None, mask_stop=True)
        for k in range(3):
            rows.append(be.slow_step(frame, 70 + k))
            frame, _ = be.frame_step_greedy(None, mask_stop=True)
        frames = [frame]
        for _ in range(70):
            frame, _ = be.frame_step_greedy(frame, mask_stop=True)
            frames.append(frame)
        outs.append((rows, np.array(frames), be.decode_greedy(20, mask_stop=True)))
        be.close()
    (ra, fa, da), (rb, fb, db) = outs
    assert np.array_equal(fa, fb) and np.array_equal(da, db)
    # a bf16 cache rounds a key that moved by an ulp to the next step: 2^-8 of one element
    tol = 1e-3 if kv == SX_DTYPE_F32 else 2e-2
    for a, b in zip(ra, rb):
        assert np.max(np.abs(a.semantic_logits - b.semantic_logits)) <= tol
        assert np.max(np.abs(a.hidden - b.hidden)) <= 50 * tol


def test_batch_of_uneven_sequences_shares_the_pool(tiny):
    """Four sequences whose pages would not fit side by side at max_ctx each."""
    m, _ = tiny
    Ts = [5, 200, 63, 64]
    prompts = [prompt_for(TINY_S2, T, seed=20 + T) for T in Ts]
    need = sum(pages(T + 30) for T in Ts)
    a = sx.B200DualAr(m, max_ctx=1024, max_batch=4)
    b = sx.B200DualAr(m, max_ctx=1024, max_batch=4, pool_pages=need)
    sa, sb = a.prefill_batch(prompts), b.prefill_batch(prompts)
    assert np.max(np.abs(sa.semantic_logits - sb.semantic_logits)) <= 1e-3
    assert b.pool_free() == need - sum(pages(T) for T in Ts)
    fa, fb = a.decode_greedy_batch(4, 30, mask_stop=True), b.decode_greedy_batch(4, 30, mask_stop=True)
    assert all(np.array_equal(x, y) and len(y) == 30 for x, y in zip(fa, fb))
    assert b.pool_free() == 0
    # some of the batch idle, then all again: an idle sequence's place is written over
    b.reset()
    a.reset()
    a.prefill_batch(prompts), b.prefill_batch(prompts)
    frames = [list(x[0]) for x in fa]
    for active in ([1, 0, 1, 1], [0, 0, 1, 0], [1, 1, 1, 1]):
        la, lb = a.slow_step_batch(frames, active), b.slow_step_batch(frames, active)
        assert np.max(np.abs(la.semantic_logits - lb.semantic_logits)) <= 1e-3
    a.close()
    b.close()


def test_pool_runs_out_and_comes_back(tiny):
    m, _ = tiny
    be = sx.B200DualAr(m, max_ctx=512, max_batch=2, pool_pages=3)
    with pytest.raises(sx.SyrinxError) as e:
        be.prefill(prompt_for(TINY_S2, 193, seed=1))
    assert e.value.code == -7 and be.pool_free() == 3
    be.prefill(prompt_for(TINY_S2, 192, seed=1))
    assert be.pool_free() == 0
    with pytest.raises(sx.SyrinxError) as e:
        be.slow_step(be.frame_step_greedy(None, mask_stop=True)[0], 192)
    assert e.value.code == -7
    assert len(be.decode_greedy(5, mask_stop=True)) == 0
    be.reset()
    assert be.pool_free() == 3
    first = be.prefill(prompt_for(TINY_S2, 100, seed=2)).semantic_logits
    frames = be.decode_greedy(500, mask_stop=True)
    assert len(frames) == 92 and be.pool_free() == 0  # to the last position of the third page
    be.reset()
    assert np.array_equal(be.prefill(prompt_for(TINY_S2, 100, seed=2)).semantic_logits, first)
    assert np.array_equal(be.decode_greedy(92, mask_stop=True), frames)
    # a refused batch leaves the pages that are free as they were
    be.reset()
    with pytest.raises(sx.SyrinxError):
        be.prefill_batch([prompt_for(TINY_S2, 100, seed=2), prompt_for(TINY_S2, 130, seed=3)])
    be.reset()
    assert be.pool_free() == 3
    be.close()


def test_stopped_sequences_and_sampled_frames(tiny):
    """Without masking, sequences may stop inside a loop; the loop's draws equal a static session's."""
    m, _ = tiny
    prompts = [prompt_for(TINY_S2, T, seed=40 + T) for T in (64, 10, 127)]
    a = sx.B200DualAr(m, max_ctx=256, max_batch=3)
    b = sx.B200DualAr(m, max_ctx=256, max_batch=3, pool_pages=9)
    a.prefill_batch(prompts), b.prefill_batch(prompts)
    for n in (40, 1, 25):
        fa, fb = a.decode_greedy_batch(3, n), b.decode_greedy_batch(3, n)
        assert all(np.array_equal(x, y) for x, y in zip(fa, fb))
    a.reset(), b.reset()
    a.prefill(prompts[0]), b.prefill(prompts[0])
    p = sx.SamplingParams()
    assert np.array_equal(a.decode_sample(30, 5, p), b.decode_sample(30, 5, p))
    a.close()
    b.close()


def test_plain_lm_with_bias_and_half_head_rotation():
    cfg = shrink(COSYVOICE2_LM, 2)
    m = sx.Model(cfg, sx.synth_blob(cfg, SX_DTYPE_Q8_0, seed=5), device=0)
    a, b = sx.B200DualAr(m, max_ctx=300), sx.B200DualAr(m, max_ctx=300, pool_pages=5)
    ids = prompt_for(cfg, 90, seed=1)[0]
    la, lb = a.lm_step_tokens(ids), b.lm_step_tokens(ids)
    assert np.max(np.abs(la - lb)) <= 1e-3
    for k in range(3):
        la, lb = a.lm_step_tokens([int(ids[k])]), b.lm_step_tokens([int(ids[k])])
        assert np.max(np.abs(la - lb)) <= 1e-3
    emb = np.random.default_rng(0).normal(0, 0.02, (70, cfg.slow.dim)).astype(np.float32)
    assert np.max(np.abs(a.lm_step_embeds(emb) - b.lm_step_embeds(emb))) <= 1e-3
    assert np.array_equal(a.decode_greedy(40, mask_stop=True), b.decode_greedy(40, mask_stop=True))
    for x in (a, b):
        x.close()
    m.close()


def test_long_synthetic_context(tiny):
    """A context that spreads over every SM, filled as if prefilled; both sessions hold the same values."""
    m, _ = tiny
    a = sx.B200DualAr(m, max_ctx=20000)
    b = sx.B200DualAr(m, max_ctx=20000, pool_pages=pages(19990))
    prompt = prompt_for(TINY_S2, 10, seed=9)
    outs = []
    for be in (a, b):
        be.fill_kv_synthetic(19960, seed=4)
        outs.append((be.prefill(prompt).semantic_logits, be.decode_greedy(20, mask_stop=True)))
    assert np.max(np.abs(outs[0][0] - outs[1][0])) <= 1e-3
    assert np.array_equal(outs[0][1], outs[1][1])
    assert b.pool_free() == 0
    a.close()
    b.close()


def test_refusals(tiny):
    m, _ = tiny
    for bad in (dict(pool_pages=-1), dict(pool_pages=1 << 25), dict(pool_pages=4, max_batch=9)):
        with pytest.raises(sx.SyrinxError):
            sx.B200DualAr(m, max_ctx=64, **bad)
    be = sx.B200DualAr(m, max_ctx=64)
    with pytest.raises(sx.SyrinxError):
        be.pool_free()
    be.close()
