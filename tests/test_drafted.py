"""Drafted greedy decoding (mw_decode_drafted): refusals on the CPU where no context is needed, and on the GPU the ids of greedy
decoding whatever the drafts are, in fewer passes when they are good."""
import numpy as np
import pytest

import manual_whisper_amd as mw
from manual_whisper_amd import synth
from manual_whisper_amd.decode_options import DecodeOptions, synthetic_options
from oracle.whisper_ref import WhisperOracle, log_mel


def test_a_null_context_is_refused():
    from manual_whisper_amd import _lib
    assert _lib.load().mw_decode_drafted(None, 1, 4, None, None, 0, 1, None, None) == -1


def _same_up_to_near_ties(got, want, orc, enc, opts, gap=2e-2):
    """ids equal; where they part, the oracle's two best logits at that place are within an fp16 rounding of each other."""
    for b in range(got.shape[0]):
        differ = np.nonzero(got[b] != want[b])[0]
        if len(differ) == 0:
            continue
        n = int(differ[0])
        seq = np.asarray(list(opts.prompt) + want[b, :n].tolist(), np.int32)[None]
        row = orc.forced_logits(enc[b:b + 1], seq)[0, -1].astype(np.float64)
        sup = set(opts.effective_suppress()) | (set(opts.begin_suppress) if n == 0 else set())
        row[list(sup)] = -np.inf
        assert abs(row[got[b, n]] - row[want[b, n]]) < gap, (b, n)


def _engine(name, max_batch, n, weight_format="f16", kv_format="f16"):
    from manual_whisper_amd.engine import Engine
    dims = mw.get_dims(name)
    w = synth.make_weights_np(dims, 1234)
    pcm = synth.make_pcm_np(n, seed=1)
    eng = Engine(dims, device=0, max_batch=max_batch, weight_format=weight_format, kv_format=kv_format)
    eng.load_weights(w)
    eng.logmel(pcm, want_output=False)
    eng.encode(n, want_output=False)
    return dims, w, pcm, eng


@pytest.mark.gpu
@pytest.mark.parametrize("name,max_new", [("micro", 40), ("tiny", 24)])
def test_drafts_change_the_passes_and_not_the_ids(name, max_new):
    n = 3
    dims, w, pcm, eng = _engine(name, 48, n)
    orc = WhisperOracle(dims, w)
    enc = orc.encode(log_mel(pcm, dims.n_mels))
    rng = np.random.default_rng(0)
    base = synthetic_options(dims, max_new=max_new)
    for prompt in (base.prompt, tuple(base.prompt) + tuple(int(x) for x in rng.integers(5, dims.vocab // 2, 37))):
        opts = DecodeOptions(prompt=prompt, suppress=base.suppress, begin_suppress=base.begin_suppress, eot=base.eot, max_new=max_new)
        eng.set_decode_options(opts)
        want, want_len, _ = eng.decode_greedy(n)
        text = [want[b, :want_len[b]].tolist() + [opts.eot] * int(want_len[b] < max_new) for b in range(n)]
        wrong = [[(x + 1) % 500 for x in t] for t in text]
        gaps = [t[:3] + t[4:9] + [7] + t[9:] for t in text]                     # a word left out, a word too many
        noise = [rng.integers(0, dims.vocab, 60).tolist() for _ in range(n)]
        for nodes in (2, 5, 8, 16):
            for drafts, passes in (([[] for _ in range(n)], None), ([[t] for t in text], -(-max(len(t) for t in text) // nodes) + 1),
                                   ([[x] for x in wrong], None), ([[x] for x in gaps], None),
                                   ([[a, b, c] for a, b, c in zip(noise, gaps, text)], None), ([[text[0]], [], [noise[2], text[2]]], None)):
                got, got_len = eng.decode_drafted(n, drafts, nodes)
                _same_up_to_near_ties(got, want, orc, enc, opts)
                if (got == want).all():
                    assert (got_len == want_len).all()
                    steps = eng.stage_ms()["decode_steps"]
                    assert steps <= max_new
                    if passes is not None:      # all of the draft is taken, `nodes` tokens a pass; the poll sees the end a little later
                        assert steps <= passes + 2 * 4, (steps, passes)
    eng.close()


@pytest.mark.gpu
@pytest.mark.parametrize("nodes,n_prompt,max_new", [(64, 1, 40), (33, 1, 1), (64, 4, 2), (17, 2, 60)])
def test_widest_trees_and_shortest_prompts(nodes, n_prompt, max_new):
    """Trees over two mask words, a prompt of one token, decodes of one and two tokens; drafts right, interleaved and of several kinds."""
    n = 2
    dims, w, pcm, eng = _engine("micro", 2 * nodes, n)
    orc = WhisperOracle(dims, w)
    enc = orc.encode(log_mel(pcm, dims.n_mels))
    base = synthetic_options(dims, max_new=max_new)
    opts = DecodeOptions(prompt=tuple(base.prompt)[:n_prompt], suppress=base.suppress, begin_suppress=base.begin_suppress, eot=base.eot, max_new=max_new)
    eng.set_decode_options(opts)
    want, want_len, _ = eng.decode_greedy(n)
    text = [want[b, :want_len[b]].tolist() for b in range(n)]
    rng = np.random.default_rng(nodes)
    noise = [[rng.integers(0, dims.vocab, 50).tolist() for _ in range(5)] for _ in range(n)]
    for drafts in ([[t] for t in text], [[t, t[1:], t[2:]] + x for t, x in zip(text, noise)], noise, [[], [text[1]]]):
        got, got_len = eng.decode_drafted(n, drafts, nodes)
        _same_up_to_near_ties(got, want, orc, enc, opts)
        if (got == want).all():
            assert (got_len == want_len).all() and eng.stage_ms()["decode_steps"] <= max_new
    eng.close()


@pytest.mark.gpu
def test_a_decode_without_graphs_and_one_after_other_kinds_agree():
    """The same call with and without captured passes, between greedy, beam and sampled decodes that use the same memory."""
    n = 2
    dims, w, pcm, eng = _engine("tiny", 24, n)
    opts = synthetic_options(dims, max_new=16)
    eng.set_decode_options(opts)
    want, want_len, _ = eng.decode_greedy(n)
    drafts = [[want[b, :9].tolist(), want[1 - b].tolist()] for b in range(n)]
    first, first_len = eng.decode_drafted(n, drafts, 12)
    eng.set_option("graph", 0)
    plain, plain_len = eng.decode_drafted(n, drafts, 12)
    assert (first == plain).all() and (first_len == plain_len).all()
    eng.set_option("graph", 1)
    for _ in range(3):
        eng.decode_beam(n, 3)
        eng.decode_sample(n, 0.7, best_of=2, seed=3)
        again, _ = eng.decode_drafted(n, drafts, 12)
        assert (again == first).all()
        greedy, greedy_len, _ = eng.decode_greedy(n)
        assert (greedy == want).all() and (greedy_len == want_len).all()
    eng.set_decode_options(synthetic_options(dims, max_new=7))                  # a shorter limit: captured passes of the old one stay out
    short, short_len = eng.decode_drafted(n, drafts, 12)
    assert short.shape == (n, 7) and (short == first[:, :7]).all() and (short_len == np.minimum(first_len, 7)).all()
    eng.close()


@pytest.mark.gpu
@pytest.mark.parametrize("weights,kv", [("fp8", "f16"), ("fp8", "fp8")])
def test_fp8_engines(weights, kv):
    n = 2
    dims, w, pcm, eng = _engine("tiny", 32, n, weights, kv)
    opts = synthetic_options(dims, max_new=16)
    eng.set_decode_options(opts)
    want, want_len, _ = eng.decode_greedy(n)
    orc = WhisperOracle(dims, w, weight_format="fp8")
    enc = orc.encode(log_mel(pcm, dims.n_mels))
    got, got_len = eng.decode_drafted(n, [[want[b].tolist()] for b in range(n)], 8)
    _same_up_to_near_ties(got, want, orc, enc, opts, gap=0.1)                   # row-quantised activations: a wider near-tie
    eng.close()


@pytest.mark.gpu
def test_forks_with_a_small_cache_and_end_of_text():
    """Recordings x nodes sequences on a fork whose cross-attention cache holds the recordings only; recordings that end early."""
    n = 4
    dims, w, pcm, eng = _engine("micro", n, n)
    base = synthetic_options(dims, max_new=30)
    child = eng.fork(max_batch=n * 6, cache_sequences=n)
    child.encode_into(pcm, child, 0)
    child.set_encoded(n)
    eng.set_decode_options(base)
    ids, _, _ = eng.decode_greedy(n)
    # end-of-text = a token that greedy decoding reaches: some recordings end there
    eot = int(ids[1, 5])
    opts = DecodeOptions(prompt=base.prompt, suppress=base.suppress, begin_suppress=base.begin_suppress, eot=eot, max_new=30)
    eng.set_decode_options(opts)
    child.set_decode_options(opts)
    want, want_len, _ = eng.decode_greedy(n)
    assert (want_len < 30).any()
    for drafts in ([[ids[b].tolist()] for b in range(n)], [[] for _ in range(n)]):
        got, got_len = child.decode_drafted(n, drafts, 6)
        orc = WhisperOracle(dims, w)
        _same_up_to_near_ties(got, want, orc, orc.encode(log_mel(pcm, dims.n_mels)), opts)
        if (got == want).all():
            assert (got_len == want_len).all()
    eng.close()


@pytest.mark.gpu
def test_arguments_are_checked():
    from manual_whisper_amd.engine import EngineError
    dims, w, pcm, eng = _engine("micro", 16, 2)
    opts = synthetic_options(dims, max_new=8)
    with pytest.raises(EngineError):
        eng.decode_drafted(2, [[], []], 4)                    # no options yet
    eng.set_decode_options(opts)
    good = [[[5, 6]], [[7]]]
    eng.decode_drafted(2, good, 8)
    for n, drafts, nodes in ((2, good, 1), (2, good, 65), (2, good, 9), (1, good[:1], 4), (3, good + [[]], 4), (2, good[:1], 4),
                             (2, [[[5, -1]], []], 4), (2, [[[dims.vocab]], []], 4), (2, [[[1]] * 9, []], 4), (2, [[[1] * 1001], []], 4)):
        with pytest.raises(EngineError):
            eng.decode_drafted(n, drafts, nodes)
    eng.decode_drafted(2, good, 8)
    eng.close()


# Polls of "all have ended" are four passes apart and one behind: up to eight passes more than the text needs.
POLLS = 2 * 4


def _passes(lens, nodes, max_new):
    """Passes for texts that drafts have right: the prompt's, which yields a token, and one per `nodes` tokens."""
    return 1 + max(-(-(min(n + 1, max_new) - 1) // nodes) for n in lens)


@pytest.mark.gpu
@pytest.mark.parametrize("name,weights,kv,nodes,max_new", [("tiny", "fp8", "f16", 8, 48), ("tiny", "fp8", "fp8", 8, 48), ("micro", "f16", "f16", 64, 60),
                                                           ("micro", "f16", "f16", 33, 60), ("micro", "f16", "f16", 17, 60)])
def test_right_drafts_are_accepted(name, weights, kv, nodes, max_new):
    """Drafts that are what drafted decoding itself returns take `nodes` tokens a pass, in fp8 engines and trees over two mask words too."""
    n = 2
    dims, w, pcm, eng = _engine(name, n * nodes, n, weights, kv)
    eng.set_decode_options(synthetic_options(dims, max_new=max_new))
    text, lens = eng.decode_drafted(n, [[] for _ in range(n)], nodes)
    for _ in range(3):          # near-equal logits may fall differently in another grouping: what was decoded becomes the next draft
        got, got_len = eng.decode_drafted(n, [[text[b, :lens[b]].tolist()] for b in range(n)], nodes)
        same = (got == text).all()
        text, lens = got, got_len
        if same:
            break
    assert same and eng.stage_ms()["decode_steps"] <= _passes(lens, nodes, max_new) + POLLS < max_new
    eng.close()


@pytest.mark.gpu
def test_right_drafts_are_accepted_up_to_the_end_of_text():
    n, nodes, max_new = 3, 6, 60
    dims, w, pcm, eng = _engine("micro", n * nodes, n)
    base = synthetic_options(dims, max_new=max_new)
    eng.set_decode_options(base)
    ids, _, _ = eng.decode_greedy(n)
    eng.set_decode_options(DecodeOptions(prompt=base.prompt, suppress=base.suppress, begin_suppress=base.begin_suppress, eot=int(ids[1, 20]),
                                         max_new=max_new))
    want, want_len, _ = eng.decode_greedy(n)
    assert want_len[1] <= 20
    eot = [int(ids[1, 20])]
    got, got_len = eng.decode_drafted(n, [[want[b, :want_len[b]].tolist() + eot * int(want_len[b] < max_new)] for b in range(n)], nodes)
    assert (got == want).all() and (got_len == want_len).all()
    assert eng.stage_ms()["decode_steps"] <= _passes(want_len, nodes, max_new) + POLLS < max_new
    eng.close()
