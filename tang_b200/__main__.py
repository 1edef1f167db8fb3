"""Command line: ``python -m tang_b200 generate --model DIR --prompt 1,2,3``, ``python -m tang_b200 score --model DIR --tokens 1,2,3`` and
``python -m tang_b200 trace ...``."""
from __future__ import annotations

import argparse
import sys


def generate(argv) -> int:
    ap = argparse.ArgumentParser(prog="tang_b200 generate", description="Generates token ids from prompts of token ids.")
    ap.add_argument("--model", required=True, help="folder with config.json and model.safetensors")
    ap.add_argument("--prompt", action="append", required=True, help="comma-separated token ids; may be repeated (one batch)")
    ap.add_argument("--max-new", type=int, default=32)
    ap.add_argument("--dtype", default="bfloat16", choices=["bfloat16", "float32"])
    ap.add_argument("--temperature", type=float, default=0.0, help="0: greedy")
    ap.add_argument("--top-k", type=int, default=0)
    ap.add_argument("--top-p", type=float, default=1.0)
    ap.add_argument("--repetition-penalty", type=float, default=1.0)
    ap.add_argument("--seed", type=int, default=42)
    ap.add_argument("--logprobs", action="store_true", help="below each line its tokens' log probabilities")
    ap.add_argument("--device", type=int, default=0)
    args = ap.parse_args(argv)

    from . import _build, _lib

    _lib.load(_build.ensure("dense"))
    from .device import QuantComputeDevice, SamplerConfig
    from .registry import DTYPES, load_model

    prompts = [[int(t) for t in p.split(",")] for p in args.prompt]
    dev = QuantComputeDevice(args.device)
    model = load_model(dev, args.model, DTYPES[args.dtype], max_slots=len(prompts), max_seq=max(map(len, prompts)) + args.max_new)
    cfg = SamplerConfig(args.temperature, args.top_k, args.top_p, args.repetition_penalty)
    tokens, rates = model.generate(prompts, args.max_new, cfg, args.seed, logprobs=True) if args.logprobs else (
        model.generate(prompts, args.max_new, cfg, args.seed), None)
    for i, row in enumerate(tokens):
        print(",".join(str(int(t)) for t in row))
        if rates is not None:
            print(",".join(f"{x:.6f}" for x in rates[i]))
    model.destroy()
    dev.close()
    return 0


def score(argv) -> int:
    ap = argparse.ArgumentParser(prog="tang_b200 score", description="Log probability of every token but the first after those before it.")
    ap.add_argument("--model", required=True, help="folder with config.json and model.safetensors")
    ap.add_argument("--tokens", action="append", required=True, help="comma-separated token ids; may be repeated")
    ap.add_argument("--dtype", default="bfloat16", choices=["bfloat16", "float32"])
    ap.add_argument("--device", type=int, default=0)
    args = ap.parse_args(argv)

    from . import _build, _lib

    _lib.load(_build.ensure("dense"))
    from .device import QuantComputeDevice
    from .engine import Engine
    from .registry import DTYPES, load_model

    texts = [[int(t) for t in p.split(",")] for p in args.tokens]
    dev = QuantComputeDevice(args.device)
    model = load_model(dev, args.model, DTYPES[args.dtype], max_slots=len(texts), max_seq=max(map(len, texts)))
    for row in Engine(model).score(list(enumerate(texts))):
        print(",".join(f"{x:.6f}" for x in row["logprobs"]))
    model.destroy()
    dev.close()
    return 0


def main(argv=None) -> int:
    argv = sys.argv[1:] if argv is None else argv
    if argv and argv[0] == "generate":
        return generate(argv[1:])
    if argv and argv[0] == "score":
        return score(argv[1:])
    if argv and argv[0] == "trace":
        from .trace import main as trace

        return trace(argv[1:])
    print(__doc__, file=sys.stderr)
    return 2


if __name__ == "__main__":
    sys.exit(main())
