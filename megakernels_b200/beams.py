"""Beam search over the sequences of a generator.

No counterpart in the reference, which decodes greedily (megakernels/generators.py:121-163).  One
loop for both families: a generator says how many sequences it has (``beam_limits``), puts prompts into
them (``start_beams``), advances all of them by a token (``step_beams``) and lets every sequence go on from
another one's cache or state (``reorder_beams``).  What follows a step - the best continuations of a
prompt's beams, the tables of tokens, ended beams - stays on the device; the loop reads nothing back
but, now and then, whether all beams have ended.
"""

from __future__ import annotations

from dataclasses import dataclass

import torch
from torch import Tensor

from megakernels_b200.mk import get_mk_module


@dataclass
class BeamResult:
    """Of every prompt its beams, best first.  A beam that has ended has ``eos`` in ``tokens`` from its end on."""

    tokens: Tensor  # int64 [prompts, beams, tokens]
    lengths: Tensor  # int64 [prompts, beams]: tokens up to the first eos, that included
    scores: Tensor  # float32 [prompts, beams]: sums of log-probabilities
    ranks: Tensor  # float32 [prompts, beams]: scores / lengths ** length_penalty, what beams are ordered by


def beam_search(gen, prompts, beams: int | None = None, ntok: int = 100, *, eos: int | None = None, length_penalty: float = 0.0,
                check_interval: int = 16) -> BeamResult:
    """Up to ``ntok`` tokens behind each prompt: one tensor of token ids, a list of them, or a matrix with a prompt per row.

    At every step the ``beams`` best of a prompt's beams x vocabulary continuations go on (equal ones: the lowest
    beam, then the lowest token).  A beam that takes ``eos`` has ended: it competes with its score and is not
    continued.  In the end beams are ordered by score / length ** ``length_penalty``.  Every ``check_interval`` steps
    the host looks whether all beams have ended.
    """
    if isinstance(prompts, Tensor):
        prompts = list(prompts) if prompts.ndim == 2 else [prompts]
    if any(p.numel() != max(p.shape, default=1) for p in prompts):
        raise ValueError("a prompt is one row of token ids")
    prompts = [p.reshape(-1) for p in prompts]
    sequences, positions = gen.beam_limits()
    beams = sequences // max(len(prompts), 1) if beams is None else beams
    ops = get_mk_module(name="mk_sequences")
    if not prompts or any(p.numel() == 0 for p in prompts):
        raise ValueError("beam search needs prompts of a token and more")
    if not 1 <= beams <= min(ops.MAX_BEAMS, gen.model.config.vocab_size) or len(prompts) * beams > sequences:
        raise ValueError(f"{len(prompts)} prompts with {beams} beams each, of {sequences} sequences in all (at most {ops.MAX_BEAMS} beams)")
    if check_interval < 1:
        raise ValueError(f"a look at the beams every {check_interval} steps")
    if ntok < 1 or max(p.numel() for p in prompts) + ntok - 1 > positions:
        raise ValueError(f"{ntok} tokens behind a prompt of {max(p.numel() for p in prompts)}: there are {positions} positions")
    first, rows = min(p.numel() for p in prompts), len(prompts) * beams
    if eos is not None and not 0 <= eos < gen.model.config.vocab_size:
        raise ValueError(f"eos {eos} outside a vocabulary of {gen.model.config.vocab_size}")
    try:
        logits = gen.start_beams(prompts, beams)
        device = logits.device
        lengths = torch.tensor([p.numel() for p in prompts], dtype=torch.int32, device=device).repeat_interleave(beams)
        table = torch.zeros(rows, ntok, dtype=torch.int64, device=device)
        count = torch.ones(rows, dtype=torch.int64, device=device)
        # (each prompt's best first tokens: its beams have one past in common)
        scores, _, tokens, done = ops.beam_select(logits, beams=1, k=beams, eos=eos)
        table[:, 0] = tokens.view(-1)
        n = 1
        while n < ntok:
            if eos is not None and n % check_interval == 0 and bool((done != 0).all()):
                break
            logits = gen.step_beams(tokens.view(-1), lengths)
            lengths = lengths + 1
            over = done.view(-1)
            scores, parents, tokens, done = ops.beam_select(logits, scores, beams=beams, k=beams, done=done if eos is not None else None, eos=eos)
            chosen = parents.view(-1)
            gen.reorder_beams(chosen, first, lengths)
            table = table[chosen]
            table[:, n] = tokens.view(-1)
            count = count[chosen] + (over[chosen] == 0)
            n += 1
    finally:
        gen.end_beams()
    shape = (len(prompts), beams)
    count = count.view(shape)
    ranks = scores / count.float() ** length_penalty
    order = torch.sort(ranks, dim=1, descending=True, stable=True).indices
    pick = lambda t: t.gather(1, order)  # noqa: E731
    tokens = table[:, :n].view(*shape, n).gather(1, order.unsqueeze(-1).expand(-1, -1, n))
    return BeamResult(tokens, pick(count), pick(scores), pick(ranks))
