"""The decoder's batch over a paged cache, and scaled rotary positions, against the numpy oracle."""
import dataclasses

import numpy as np
import pytest

import kv_ref
from litenn_b200 import capi, synth
from litenn_b200 import llama as ll

pytestmark = pytest.mark.gpu

SMALL = ll.LlamaSpec(n_layers=2, d_model=512, n_heads=8, n_kv_heads=2, head_dim=64, ffn=768, vocab=1024,
                     linear_fmt=synth.Q4_K, down_fmt=synth.Q6_K, embd_fmt=synth.Q6_K, max_seq=200, max_prefill=160)
PARTIAL = ll.LlamaSpec(n_layers=2, d_model=256, n_heads=2, n_kv_heads=1, head_dim=128, ffn=512, vocab=512,
                       linear_fmt=synth.Q8_0, embd_fmt=synth.Q6_K, max_seq=64, max_prefill=32,
                       rope_dim=64, unit_norms=False, tied_output=True)


@pytest.fixture(scope="module")
def stream(qmm_lib):
    import torch
    assert torch.cuda.is_available()
    torch.cuda.set_device(0)
    s = torch.cuda.Stream()
    yield s.cuda_stream
    del s


def stored_like(fmt, head_dim):
    """What takes the place of the oracle's rounding of cached rows to fp16."""
    def rounding(x):
        x = np.asarray(x, dtype=np.float32)
        return kv_ref.stored(x.reshape(len(x), -1, head_dim), fmt).astype(np.float32).reshape(x.shape)
    return rounding


def apart(a, e):
    """2-norm of the difference over the expected vector's."""
    return float(np.linalg.norm(np.asarray(a, np.float64) - e) / np.linalg.norm(np.asarray(e, np.float64)))


# Both sides round activations to bf16 at the same points; sums in another order flip a few of those roundings, which moves the
# logits by some 1e-5 of their norm (narrow models, contiguous cache).  Keys and values that move by that much land on another
# quant about once in (step / 1e-5 of a value): one value in 10^3 of Q4_0's steps of 1/8, off by a step, is 1/8 / 10^1.5 = 4e-3
# of a row; Q8_0's steps are a sixteenth.  Twice that, and the same for fp16 as for Q8_0.
APART = {capi.KV_F16: 1e-3, capi.Q8_0: 1e-3, capi.Q4_0: 1e-2}


def against_oracles(monkeypatch, stream, spec, fmt, page, lens, steps, scaling=None, factors=None):
    from oracle import llama_ref
    monkeypatch.setattr(llama_ref, "_fp16", stored_like(fmt, spec.head_dim))
    model = ll.LlamaModel(spec, stream=stream, seed=0)
    freq = None
    if scaling is not None or factors is not None:
        model.set_rope_scaling(scaling, factors)
        freq, gain = capi.rope_frequencies(spec.rdim, spec.rope_theta, factors, scaling)
    model.batch_create_paged(len(lens), steps, fmt, page)
    want = np.zeros((steps, len(lens)), dtype=np.int64)
    excused = [steps] * len(lens)
    matters = []
    for b, n in enumerate(lens):
        ref = llama_ref.LlamaOracle(spec, seed=0)
        if freq is not None:
            ang = np.arange(spec.max_seq)[:, None] * freq
            ref.cos, ref.sin = (np.cos(ang) * gain).astype(np.float32), (np.sin(ang) * gain).astype(np.float32)
        prompt = synth.make_token_ids(n, spec.vocab, seed=11 + b, name="paged-prompt")
        cur = ref.prefill(prompt)
        got = model.batch_prefill(b, prompt)
        logits = model.last_logits()
        off = apart(logits, ref.last_logits)
        assert off <= APART[fmt], (b, off)
        if freq is not None:  # a model that ignored the scaling would be as far off as the unscaled oracle is
            plain = llama_ref.LlamaOracle(spec, seed=0)
            plain.prefill(prompt)
            matters.append(apart(plain.last_logits, ref.last_logits))
            assert off <= matters[-1] / 3 or matters[-1] < 3 * APART[fmt]   # some prompts' attention is all on one token
        gap, scale = ref.top2_gap()
        assert got == cur or gap <= 2e-2 * scale
        cur = got
        for s in range(steps):
            cur = ref.decode_step(cur)
            want[s, b] = cur
            gap, scale = ref.top2_gap()
            if gap <= 1e-2 * scale:
                excused[b] = min(excused[b], s)
    assert freq is None or max(matters) >= 3 * APART[fmt], matters
    got = model.batch_decode(steps)
    assert capi.kernel_status(0) == 0
    for b in range(len(lens)):
        assert got[:excused[b], b].tolist() == want[:excused[b], b].tolist(), b
    assert sum(excused) >= steps * len(lens) // 2
    model.close()


@pytest.mark.parametrize("fmt", [capi.KV_F16, capi.Q8_0, capi.Q4_0])
@pytest.mark.parametrize("spec,lens,page", [(SMALL, [5, 150, 31], 16), (PARTIAL, [9, 30], 64)], ids=["grouped", "partial-rope"])
def test_paged_batch_matches_one_oracle_per_sequence(monkeypatch, stream, spec, lens, page, fmt):
    against_oracles(monkeypatch, stream, spec, fmt, page, lens, 8)


@pytest.mark.parametrize("scaling,factors", [(capi.RopeScaling(capi.ROPE_SCALE_YARN, 4.0, 32, 32, 1), False),
                                             (capi.RopeScaling(capi.ROPE_SCALE_LINEAR, 2.0, 0, 0, 0), True), (None, True)],
                         ids=["yarn", "linear+factors", "factors"])
def test_paged_batch_with_scaled_positions(monkeypatch, stream, scaling, factors):
    spec = SMALL
    f = np.linspace(1, 4, spec.rdim // 2).astype(np.float32) if factors else None
    against_oracles(monkeypatch, stream, spec, capi.Q8_0, 32, [40, 7, 150], 6, scaling, f)


def test_scaled_positions_of_the_single_sequence(stream):
    """prefill and decode over the contiguous cache follow set_rope_scaling too."""
    from oracle.llama_ref import LlamaOracle
    spec = SMALL
    scaling = capi.RopeScaling(capi.ROPE_SCALE_YARN, 4.0, 32, 32, 1)
    model = ll.LlamaModel(spec, stream=stream, seed=0)
    prompt = synth.make_token_ids(40, spec.vocab, seed=2, name="scaled")
    plain_token = model.prefill(prompt)
    plain = model.last_logits()
    with pytest.raises(capi.QmmError):
        model.set_rope_scaling(scaling)             # the cache holds tokens
    model.reset()
    model.set_rope_scaling(scaling)
    ref = LlamaOracle(spec, seed=0)
    freq, gain = capi.rope_frequencies(spec.rdim, spec.rope_theta, None, scaling)
    ang = np.arange(spec.max_seq)[:, None] * freq
    ref.cos, ref.sin = (np.cos(ang) * gain).astype(np.float32), (np.sin(ang) * gain).astype(np.float32)
    ref.prefill(prompt)
    model.prefill(prompt)
    off = apart(model.last_logits(), ref.last_logits)
    assert off <= 1e-3 and off <= apart(plain, ref.last_logits) / 3      # a model that ignored the scaling gives `plain`
    cur = 3
    for _ in range(3):
        ref.decode_step(cur)
        model.step_host(cur)
        assert apart(model.last_logits(), ref.last_logits) <= 1e-3
    model.reset()
    model.set_rope_scaling(None)
    assert model.prefill(prompt) == plain_token
    np.testing.assert_array_equal(model.last_logits(), plain)
    model.close()


def test_pages_are_taken_as_sequences_grow_and_come_back(stream):
    spec = SMALL
    model = ll.LlamaModel(spec, stream=stream, seed=0)
    with pytest.raises(capi.QmmError):
        model.batch_free_pages()
    for bad in ((2, 5, 9, 64), (2, 5, capi.Q4_0, 0), (2, 5, capi.Q4_0, 24), (17, 5, capi.Q4_0, 64)):
        with pytest.raises(capi.QmmError):
            model.batch_create_paged(*bad)
    model.batch_create_paged(2, 60, capi.Q4_0, 16, n_pages=6)
    assert model.batch_free_pages() == 6
    first = [model.batch_prefill(b, synth.make_token_ids(n, spec.vocab, seed=b, name="grow")) for b, n in enumerate([33, 16])]
    assert model.batch_free_pages() == 2                       # 3 and 1 pages
    a = model.batch_decode(8)                                  # 41 and 24 tokens
    assert model.batch_free_pages() == 1
    with pytest.raises(capi.QmmError) as e:
        model.batch_decode(20)                                 # 61 and 44 tokens: 4 and 3 pages, two more than held
    assert "free pages" in str(e.value) and model.batch_free_pages() == 1
    b = model.batch_decode(7)                                  # 48 and 31
    assert model.batch_free_pages() == 1
    c = model.batch_decode(1)                                  # 49 and 32: the last page
    assert model.batch_free_pages() == 0
    model.reset()
    assert model.batch_free_pages() == 6
    again = [model.batch_prefill(s, synth.make_token_ids(n, spec.vocab, seed=s, name="grow")) for s, n in enumerate([33, 16])]
    assert again == first and (model.batch_decode(16) == np.concatenate([a, b, c])).all()
    model.reset()
    with pytest.raises(capi.QmmError):
        model.batch_prefill(0, synth.make_token_ids(100, spec.vocab, seed=0, name="grow"))  # 7 pages
    model.close()


def test_paged_fp16_equals_the_contiguous_cache(stream):
    """The same prompts and steps over both kinds of cache: fp16 keys of the same values but for the last bit of a rotation."""
    spec = dataclasses.replace(SMALL, max_prefill=40)
    got = []
    for paged in (False, True):
        model = ll.LlamaModel(spec, stream=stream, seed=0)
        if paged:
            model.batch_create_paged(3, 12, capi.KV_F16, 32)
        else:
            model.batch_create(3, 12)
        for b in range(3):
            model.batch_prefill(b, synth.make_token_ids(10 + 9 * b, spec.vocab, seed=b, name="same"))
        got.append((model.last_logits(), model.batch_decode(12)))
        model.close()
    (l0, t0), (l1, t1) = got
    # The contiguous cache's prompts round probabilities to fp16, a call of so few rows over pages does not: a context value is off
    # by up to 2^-11 of sum p |v|, twice that of itself where v's signs differ.  Both are then rounded to bf16, steps of up to 2^-7:
    # a value that is off by 2^-10 lands a step away once in 8 times, a 2-norm of sqrt(2^-10 * 2^-7) = 2^-8.5 of the context, and
    # two layers' add up to 2^-8.  (A bound of 1e-3 held only as long as both sides rounded the probabilities.)
    assert apart(l1, l0) <= 2.0 ** -8
    assert (t0 == t1).mean() > 0.9
