"""A recording's results do not depend on what shares its pass: the same bits alone, in a small batch and in a large one."""
import numpy as np
import pytest

import manual_whisper_amd as mw
from manual_whisper_amd import synth
from manual_whisper_amd.decode_options import synthetic_options


@pytest.mark.gpu
@pytest.mark.parametrize("name,weights", [("micro", "f16"), ("tiny", "f16"), ("tiny", "fp8")])
def test_encoder_and_logits_alone_and_in_batches(name, weights):
    from manual_whisper_amd.engine import Engine
    dims = mw.get_dims(name)
    eng = Engine(dims, 0, 32, weight_format=weights)
    try:
        eng.load_weights(synth.make_weights_np(dims, 1234))
        mel3 = eng.logmel(synth.make_pcm_np(3, seed=1))
        eng.set_decode_options(synthetic_options(dims, max_new=6))
        alone = []
        for i in range(3):
            enc = eng.encode(1, mel=mel3[i:i + 1])
            ids, _, logits = eng.decode_greedy(1, want_logits=True)
            alone.append((enc[0].copy(), ids[0].copy(), np.array(logits)[:, 0].copy()))
        for n in (3, 17, 32):                                 # one and two row tiles of the decoder, small and large tiles of the encoder
            enc = eng.encode(n, mel=np.stack([mel3[(i * i) % 3] for i in range(n)]))
            ids, _, logits = eng.decode_greedy(n, want_logits=True)
            logits = np.asarray(logits)
            for i in range(n):
                want = alone[(i * i) % 3]
                assert np.array_equal(enc[i], want[0]), (n, i, "encoder")
                assert np.array_equal(ids[i], want[1]) and np.array_equal(logits[:, i], want[2]), (n, i, "logits")
    finally:
        eng.close()
