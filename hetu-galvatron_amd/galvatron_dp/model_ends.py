"""The ends of a model -- embedding, the last residual join and norm, head and log probabilities -- run with the package's
operators, and their times written where the strategy search reads them.

The search engine takes the time of what no layer covers from the computation profile, as
"layertype_other_bsz<B>_seq<S>": milliseconds of the forward pass for each sample (search_engine.py:123-194; the
reference's profiler fills it in from whole training runs, model_profiler.py:302-700).  On a GPU:

    python -m galvatron_dp.model_ends --hidden 4096 --vocab 128256 --seq 4096 --bsz 1 2 3 4 5 6 7 8 \\
        --profile configs/computation_profiling_bf16_llama.json

measures those entries and writes them into the file, next to the entries of the layers that are there.  An entry is of the whole
vocabulary on one GPU: the search divides it by the tensor-parallel degree itself, so a shard's time is printed only.  What is timed
are this package's operators: an entry is right for a program that runs its ends with them, and an estimate for one that does not.
"""
from __future__ import annotations

import argparse
import functools
import math
import os
from typing import NamedTuple, Optional

import torch

from . import operators as ops
from .profile_configs import read_json_config, write_json_config

__all__ = ["ModelEnds", "EndGrads", "measure", "write_profile"]

DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


class EndGrads(NamedTuple):
    loss: torch.Tensor          # [] mean of -log probability over the targets, float32
    entropy: torch.Tensor       # [...] of each place
    embedding: torch.Tensor     # [rows, hidden]
    norm: torch.Tensor          # [hidden]
    head: torch.Tensor          # [rows, hidden]
    block: torch.Tensor         # [..., hidden] what goes back into the last layer


class ModelEnds:
    """Weights of a model's ends, of the shard of the vocabulary that begins with token ``first``."""

    def __init__(self, hidden: int, vocab: int, *, dtype=torch.bfloat16, norm: str = "rms", scale: float = 1.0, shards: int = 1,
                 shard: int = 0, device="cuda", seed: int = 0):
        if vocab % shards or not 0 <= shard < shards:
            raise ValueError(f"{shards} shards do not divide {vocab} tokens, or there is no shard {shard}")
        rows = vocab // shards
        g = torch.Generator(device=device).manual_seed(seed)
        self.vocab, self.first, self.scale, self.shards = vocab, shard * rows, scale, shards

        def weights(*shape, size):
            return (torch.randn(*shape, generator=g, device=device) * size).to(dtype)

        self.table = weights(rows, hidden, size=1.0)
        self.head = weights(rows, hidden, size=hidden ** -0.5)
        self.norm = ops.Norm(norm, 1 + weights(hidden, size=0.1), weights(hidden, size=0.1) if norm == "layer" else None)

    def embed(self, tokens):
        """The residual stream that the first layer gets; of a shard, its part of the sum over the shards."""
        return ops.embedding(tokens, self.table, scale=self.scale, first=self.first)

    def logits(self, stream, block, stats: bool = False):
        """The last block's output joined with the stream and normed, through the head."""
        joined = ops.residual_norm(stream, block, pre=self.norm, stats=stats)
        return joined, torch.nn.functional.linear(joined.normed, self.head)

    def forward(self, tokens, targets, block, *, entropy: bool = False, top: int = 0):
        """From tokens to log probabilities of the targets, with ``block`` [..., hidden] in the place of what the layers add to the
        stream; of a shard, the ``LogprobParts`` to be exchanged."""
        _, logits = self.logits(self.embed(tokens), block)
        if self.shards > 1:
            return ops.logprob_parts(logits.reshape(-1, logits.shape[-1]), targets.reshape(-1), first=self.first, top=top)
        return ops.token_logprobs(logits, targets, entropy=entropy, top=top)

    def loss_and_grads(self, tokens, targets, block, into: Optional[torch.Tensor] = None, *,
                       loss_scale: Optional[float] = None) -> EndGrads:
        """The mean loss over the targets and its gradients (a whole vocabulary).  ``into`` [rows, hidden]: the table's is added to it.

        The gradients, not the loss, are multiplied by ``loss_scale`` (1 by default).  float16 needs one: the logits' gradients are
        shares of 1 over the number of targets, and what is below float16's least step, 6e-8, is lost.  The number of targets
        times some sixteen brings them into its range."""
        if self.shards > 1:
            raise ValueError("a shard's loss needs the parts of the others: forward, join_logprobs, token_logprobs_grad")
        if loss_scale is None:
            if self.table.dtype == torch.float16:
                raise ValueError("float16 needs a loss_scale: the gradient of a mean over many targets is below its least step")
            loss_scale = 1.0
        if not 0.0 < loss_scale < math.inf:
            raise ValueError(f"loss_scale must be positive and finite, not {loss_scale}")
        joined, logits = self.logits(self.embed(tokens), block, stats=True)
        row_stats = torch.empty(*targets.shape, 2, dtype=torch.float32, device=logits.device)
        r = ops.token_logprobs(logits, targets, entropy=True, row_stats=row_stats)
        held = (targets >= 0) & (targets < self.vocab)
        each = held / held.sum().clamp(min=1)
        d_logits = ops.token_logprobs_grad(logits, targets, None, each * -loss_scale, row_stats=row_stats, into=logits)
        rows, normed = (t.reshape(-1, t.shape[-1]) for t in (d_logits, joined.normed))
        d_normed, d_head = rows @ self.head, rows.t() @ normed
        g = ops.residual_norm_grad(joined.stream, block, joined.stats, d_normed.view_as(joined.normed), pre=self.norm)
        d_table = ops.embedding_grad(tokens, g.residual, self.table.shape[0], scale=self.scale, first=self.first, into=into)
        return EndGrads(-(r.logp * each).sum(), r.entropy, d_table, g.pre_weight, d_head, g.block)


def measure(ends: ModelEnds, bsz: int, seq: int, *, repeats: int = 20, backward: bool = False) -> float:
    """Milliseconds of a pass through the ends for each of ``bsz`` samples of ``seq`` tokens: the median of ``repeats``."""
    device, (rows, hidden) = ends.table.device, ends.table.shape
    g = torch.Generator(device=device).manual_seed(1)
    tokens = torch.randint(0, ends.vocab, (bsz, seq + 1), generator=g, device=device)
    block = torch.randn(bsz, seq, hidden, generator=g, device=device).to(ends.table.dtype)
    if backward:    # (float16: its range needs a scale, its time does not depend on which)
        step = functools.partial(ends.loss_and_grads, loss_scale=bsz * seq * 16.0 if ends.table.dtype == torch.float16 else None)
    else:
        step = ends.forward
    times = []
    for i in range(3 + repeats):
        begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        begin.record()
        step(tokens[:, :-1], tokens[:, 1:], block)
        end.record()
        end.synchronize()
        if i >= 3:
            times.append(begin.elapsed_time(end))
    return sorted(times)[len(times) // 2] / bsz


def write_profile(path: str, times: dict) -> dict:
    """Writes {(bsz, seq): ms} as "layertype_other_bsz<B>_seq<S>" into a computation profile, whose other entries stay."""
    config = read_json_config(path) if os.path.exists(path) else {}
    config.update({"layertype_other_bsz%d_seq%d" % key: ms for key, ms in times.items()})
    write_json_config(config, path)
    return config


def main(argv=None) -> dict:
    p = argparse.ArgumentParser(prog="python -m galvatron_dp.model_ends", description="Measures embedding, last join and norm, head and log "
                                "probabilities, for the computation profile that the strategy search reads.")
    p.add_argument("--hidden", type=int, required=True)
    p.add_argument("--vocab", type=int, required=True)
    p.add_argument("--seq", type=int, nargs="+", default=[4096])
    p.add_argument("--bsz", type=int, nargs="+", default=[1])
    p.add_argument("--precision", choices=sorted(DTYPES), default="bf16")
    p.add_argument("--norm", choices=("rms", "layer"), default="rms")
    p.add_argument("--shards", type=int, default=1, help="vocabulary-parallel degree: measures one shard, which is no entry of a profile")
    p.add_argument("--backward", action="store_true", help="prints forward and backward passes as well")
    p.add_argument("--profile", help="computation profile to write the entries into")
    a = p.parse_args(argv)
    if a.profile and a.shards > 1:
        p.error("--profile takes the time of the whole vocabulary, which the search divides by the parallel degree: not with --shards")
    ends = ModelEnds(a.hidden, a.vocab, dtype=DTYPES[a.precision], norm=a.norm, shards=a.shards)
    times = {}
    for seq in a.seq:
        for bsz in a.bsz:
            times[bsz, seq] = measure(ends, bsz, seq)
            name = "layertype_other_bsz%d_seq%d" if a.shards == 1 else "a shard of %d, bsz %%d, seq %%d" % a.shards
            line = (name + ": %.4f ms a sample") % (bsz, seq, times[bsz, seq])
            if a.backward and a.shards == 1:
                line += ", forward and backward %.4f" % measure(ends, bsz, seq, backward=True)
            print(line, flush=True)
    if a.profile:
        write_profile(a.profile, times)
    return times


if __name__ == "__main__":
    main()
