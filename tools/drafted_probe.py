#!/usr/bin/env python3
"""Times of Engine.decode_drafted beside decode_greedy: large-v3, 16 recordings of 128 tokens, random-init weights, one draft a
recording that is right by 100, 90 and 70 %.  Per (nodes, share): ms of the decode, its passes, the share of ids that equal greedy's.
Usage: python tools/drafted_probe.py [out.csv]"""
import csv
import os
import sys

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import numpy as np  # noqa: E402
import manual_whisper_amd as mw  # noqa: E402
from manual_whisper_amd import synth  # noqa: E402
from manual_whisper_amd.decode_options import whisper_options  # noqa: E402
from manual_whisper_amd.engine import Engine  # noqa: E402
import torch  # noqa: E402

N, TOKENS = 16, 128
dims = mw.get_dims("large-v3")
weights = synth.make_weights_torch(dims, 1234, device="cuda")
eng = Engine(dims, device=0, max_batch=N)
eng.load_weights(weights)
del weights
torch.cuda.empty_cache()
eng.set_decode_options(whisper_options(dims, max_new=TOKENS, suppress_eot=True))
pcm = synth.make_pcm_np(N, seed=1)
eng.logmel(pcm, want_output=False)
eng.encode(N, want_output=False)
rows = []


def report(nodes, share, same, times, passes):
    ms = sorted(times)[len(times) // 2]
    rows.append([nodes, share, f"{ms:.1f}", passes, f"{same:.4f}"])
    print(f"nodes {nodes:2d} right {share:4.0%}  {ms:7.1f} ms  {passes:4d} passes  equal ids {same:.2%}", flush=True)


times = []
for _ in range(5):
    want, _, _ = eng.decode_greedy(N)
    times.append(eng.stage_ms()["decode"])
report(1, 0.0, 1.0, times[1:], int(eng.stage_ms()["decode_steps"]))
rng = np.random.default_rng(0)
for nodes in (4, 8, 16):
    child = eng.fork(max_batch=N * nodes, cache_sequences=N)
    child.encode_into(pcm, child, 0)
    child.set_encoded(N)
    for share in (1.0, 0.9, 0.7):
        drafts = [[[int(x) if rng.random() < share else int((x + 1) % 50000) for x in want[b]]] for b in range(N)]
        times = []
        for _ in range(5):
            got, _ = child.decode_drafted(N, drafts, nodes)
            times.append(child.stage_ms()["decode"])
        report(nodes, share, (got == want).mean(), times[1:], int(child.stage_ms()["decode_steps"]))
    child.close()
eng.close()
if len(sys.argv) > 1:
    with open(sys.argv[1], "w", newline="") as f:
        w = csv.writer(f)
        w.writerow(["nodes", "right", "decode_ms", "passes", "equal_ids"])
        w.writerows(rows)
