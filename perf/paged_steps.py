"""Whole steps of PagedDecoder beside those of Transformers' static cache.

  python perf/paged_steps.py [--model llama3-8b] [--requests 32] [--low 64] [--high 2000] [--compressed]

A model of the benchmark's shapes with random weights, as it is or attached to
a NeuralZipRuntime, takes in prompts whose lengths are spread evenly from low
to high. Printed are milliseconds a step, one new token for every request: of
PagedDecoder eagerly and replayed from a HIP graph, and of the model's own
forward over a static cache that is as long for all as the longest request,
replayed from a graph (the work of a step with padded lengths, which is all
that its time depends on)."""
import argparse
import contextlib
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

import bench  # noqa: E402
from neuralzip_amd.gpu.inference import NeuralZipRuntime, export_model_for_gpu  # noqa: E402
from neuralzip_amd.gpu.paged import PagedDecoder  # noqa: E402
from neuralzip_amd.setup import NeuralZipSetup  # noqa: E402

ROOM = 128   # tokens that requests may grow by


def milliseconds(step, n):
    begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    torch.cuda.synchronize()
    begin.record()
    for _ in range(n):
        step()
    end.record()
    torch.cuda.synchronize()
    return begin.elapsed_time(end) / n


def paged(model, prompts, length):
    decoder = PagedDecoder(model, requests=len(prompts), max_length=length)
    for prompt in prompts:
        decoder.add(prompt)
    decoder.step()
    decoder.step()
    eager = milliseconds(decoder.step, 10)
    decoder.capture()
    decoder.step()
    return eager, milliseconds(decoder.step, 30)


@torch.no_grad()
def static(model, runtime, requests, length, position):
    from transformers import StaticCache
    cache = StaticCache(config=model.config, max_cache_len=length)
    token = torch.ones(requests, 1, dtype=torch.int64, device=model.device)
    at = torch.tensor([position], device=model.device)

    def step():
        out = model(input_ids=token, past_key_values=cache, cache_position=at, use_cache=True)
        return out.logits[:, -1:].argmax(-1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(), step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with runtime.graph_capture() if runtime else contextlib.nullcontext(), torch.cuda.graph(graph):
        step()
    graph.replay()
    return milliseconds(graph.replay, 20)


def main():
    parser = argparse.ArgumentParser()
    parser.add_argument("--model", choices=sorted(bench.MODELS), default="llama3-8b")
    parser.add_argument("--requests", type=int, default=32)
    parser.add_argument("--low", type=int, default=64)
    parser.add_argument("--high", type=int, default=2000)
    parser.add_argument("--compressed", action="store_true")
    args = parser.parse_args()
    model, runtime = bench.random_model(args.model, torch.device("cuda:0")), None
    print("model made", flush=True)
    if args.compressed:
        setup = NeuralZipSetup(cluster_js_threshold=0.05).build(model)
        runtime = NeuralZipRuntime.attach(model, export_model_for_gpu(model, setup), device="cuda:0")
        print("runtime attached", flush=True)
    g = torch.Generator().manual_seed(1)
    lengths = [args.low + (args.high - args.low) * i // max(args.requests - 1, 1) for i in range(args.requests)]
    prompts = [torch.randint(0, model.config.vocab_size, (n,), generator=g) for n in lengths]
    eager, replayed = paged(model, prompts, args.high + ROOM)
    print(f"{args.model}{' compressed' if runtime else ''}, {args.requests} requests of {args.low} to {args.high} tokens: "
          f"PagedDecoder {eager:.2f} ms eagerly, {replayed:.2f} from a graph", flush=True)
    padded = static(model, runtime, args.requests, args.high + ROOM, args.high)
    print(f"  static cache of {args.high + ROOM} tokens: {padded:.2f} ms from a graph", flush=True)


if __name__ == "__main__":
    main()
