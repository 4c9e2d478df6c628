"""Command line:

    python -m bitexact_llm_b200 generate --model DIR --prompt 5,17,3 [--prompt ...] [--max-new N] [--dtype D]
                                         [--temperature T] [--seed S] [--cache fp4] [--logprobs K]
    python -m bitexact_llm_b200 score --model DIR --prompt 5,17,3 [--prompt ...] [--dtype D] [--cache fp4] [--top K]
    python -m bitexact_llm_b200 trace --model DIR --dtype D --out DIR --max-tokens N   (see trace_run.py)

`generate` loads the folder through the model registry, decodes the prompts (token ids) as one batch and prints one line of
generated ids per prompt: greedy at temperature 0 (default), else the integer Gumbel sampler keyed by (seed + row, index).
With --logprobs K a line is a JSON object instead: the ids with their log probabilities, entropies, ranks and K best alternatives.
`score` prints such an object per prompt, for the prompt's own tokens from the second on. --cache fp4 keeps keys and values in 4 bits."""

import argparse
import json
import sys


def _engine(args, max_len):
    """The model of a command, its libraries built."""
    from . import build, registry
    fam = registry.family(registry.read_config(args.model))
    for target in sorted(set(fam.libraries) | {"integer"}):          # sampler and log probabilities live in the integer library
        build.build(target=target)
    return registry.load(args.model, dtype=args.dtype, max_len=max_len, cache=args.cache)


def _object(tokens, p):
    """One line of JSON: tokens and their logprobs.LogProbs; what is no number (no entry of that rank) is null."""
    num = lambda v: v if v == v and abs(v) != float("inf") else None
    top = [[[i, num(v)] for i, v in zip(*row)] for row in zip(p.top_ids.tolist(), p.top_logp.tolist())]
    return json.dumps({"tokens": tokens, "logprobs": [num(v) for v in p.logp.tolist()], "entropy": [num(v) for v in p.entropy.tolist()],
                       "rank": p.rank.tolist(), "top": top})


def score(argv):
    ap = argparse.ArgumentParser(prog="bitexact_llm_b200 score")
    ap.add_argument("--model", required=True)
    ap.add_argument("--prompt", action="append", required=True, help="token ids with commas between them")
    ap.add_argument("--dtype", default=None, help="number format of the engine (default: the model family's own)")
    ap.add_argument("--cache", default=None, help="format of keys and values: fp4 (default: the model's own)")
    ap.add_argument("--top", type=int, default=0, help="best alternatives at every place")
    args = ap.parse_args(argv)
    from .decode import score as run
    prompts = [[int(v) for v in p.split(",")] for p in args.prompt]
    eng = _engine(args, max(map(len, prompts)))
    for p, r in zip(prompts, run(eng, prompts, args.top)):
        print(_object(p[1:], r))
    return 0


def generate(argv):
    ap = argparse.ArgumentParser(prog="bitexact_llm_b200 generate")
    ap.add_argument("--model", required=True)
    ap.add_argument("--prompt", action="append", required=True, help="token ids with commas between them")
    ap.add_argument("--max-new", type=int, default=16)
    ap.add_argument("--dtype", default=None, help="number format of the engine (default: the model family's own)")
    ap.add_argument("--temperature", type=float, default=0.0)
    ap.add_argument("--seed", type=int, default=0)
    ap.add_argument("--cache", default=None, help="format of keys and values: fp4 (default: the model's own)")
    ap.add_argument("--logprobs", type=int, default=None, help="log probabilities with this many alternatives")
    args = ap.parse_args(argv)
    import torch

    from .decode import generate as run
    from .vllm_plugin.sampler import temp_ratio
    prompts = [[int(v) for v in p.split(",")] for p in args.prompt]
    longest = max(map(len, prompts))
    eng = _engine(args, longest + args.max_new)
    ids = torch.zeros(len(prompts), longest, dtype=torch.long)
    for i, p in enumerate(prompts):
        ids[i, : len(p)] = torch.tensor(p)
    tn, td = temp_ratio(args.temperature)
    toks, _, *probs = run(eng, ids, args.max_new, tn, td, seeds=[args.seed + i for i in range(len(prompts))], hashes=False,
                          lens=torch.tensor([len(p) for p in prompts]), logprobs=args.logprobs)
    for i, row in enumerate(toks.tolist()):
        print(_object(row, type(probs[0])(*(v[i] for v in probs[0]))) if probs else ",".join(map(str, row)))
    return 0


def main(argv):
    if argv[:1] == ["generate"]:
        return generate(argv[1:])
    if argv[:1] == ["score"]:
        return score(argv[1:])
    if argv[:1] == ["trace"]:
        from .trace_run import main as trace
        return trace(argv[1:])
    print(__doc__, file=sys.stderr)
    return 2


if __name__ == "__main__":
    sys.exit(main(sys.argv[1:]))
