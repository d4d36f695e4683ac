"""What 8-bit projections gain in a stack's steps: the captured decode step, the eager one and a prefill, each with projections
in bf16 and in 8 bits, without and with a norm in front of every layer.

    python perf/int8_step.py [--layers 16] [--states 1,32,64,128]

Sixteen layers of the 7B attention shape (embed 4096, 32 query and 8 KV heads of 128, a ring of 256 and two banks of 64), random
weights, Gaussian hidden states; weights and states together are larger than the L2.  Captured steps are timed on the device
with events around 100 replays after 10, the median of five; eager steps and prefills of 512 tokens by the clock between two
synchronisations, the best of five.
"""
import argparse
import os
import statistics
import sys
import time

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "coda-gqa-l_b200"))

from coda_gqa_l_b200 import CoDAGQALandmarkPerf2, CoDAStack, RMSNorm  # noqa: E402

D = 4096


def build(layers, int8, norms):
    torch.manual_seed(0)
    with torch.device("cuda"):
        made = [CoDAGQALandmarkPerf2(embed_dim=D, num_heads=32, num_kv_heads=8, window=256, num_landmarks_exact=64, num_landmarks_summary=64,
                                     rope_base=1e6, head_norm_mode="identity", rope_interleaved=False).eval().to(torch.bfloat16)
                for _ in range(layers)]
    for layer in made:
        layer.use_int8_projections = int8
    return CoDAStack(made, norms=[RMSNorm(D).to(torch.bfloat16).cuda() for _ in made] if norms else None)


def wall(call, n):
    best = float("inf")
    for _ in range(5):
        torch.cuda.synchronize()
        t = time.perf_counter()
        for _ in range(n):
            call()
        torch.cuda.synchronize()
        best = min(best, (time.perf_counter() - t) / n * 1e3)
    return best


@torch.no_grad()
def measure(layers, states, int8, norms):
    stack = build(layers, int8, norms)
    st = stack.init_states(batch_size=states, device="cuda", dtype=torch.bfloat16)
    x = torch.randn(states, 512, D, device="cuda").bfloat16() * 0.5
    token = x[:, :1].contiguous()
    stack.prefill(x, st, block_size=128, return_outputs=False)
    prefill = wall(lambda: stack.prefill(x, st, block_size=128, return_outputs=False), 1)
    for _ in range(5):
        stack.step(token, st)
    eager = wall(lambda: stack.step(token, st), 10)
    for _ in range(10):
        stack.step_graph(token, st)
    times = []
    for _ in range(5):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        for _ in range(100):
            stack.step_graph(token, st)
        b.record()
        torch.cuda.synchronize()
        times.append(a.elapsed_time(b) / 100)
    return statistics.median(times), eager, prefill


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--layers", type=int, default=16)
    ap.add_argument("--states", default="1,32,64,128")
    args = ap.parse_args()
    print("ms, bf16 -> 8 bits        captured step      eager step     prefill of 512")
    for states in map(int, args.states.split(",")):
        for norms in (False, True):
            a, b = (measure(args.layers, states, int8, norms) for int8 in (False, True))
            cells = [f"{p:7.3f} -> {q:7.3f} ({q / p - 1:+.0%})" for p, q in zip(a, b)]
            print(f"{states:4d} states{', norms' if norms else '       '}  " + "  ".join(cells), flush=True)


if __name__ == "__main__":
    main()
