"""What happens to sequences between two decoding steps: beam search's selection and the reordering of
states, the attention weight that cached keys receive, and the eviction of the others from the cache.

A case is a dict of plain values.  Kinds of cases:

* ``beam``: the best continuations of every group of beams, from the logits of a step;
* ``reorder``: every slot takes another slot's cache rows (llama caches) or its whole state (layer-list models);
* ``weights``: softmax weights of a run of queries, summed over queries and the heads that share a key;
* ``evict``: which rows of a cache stay (the first ones, the last ones, the heaviest ones), and their move to the front.

Layouts are the engines': logits ``[rows, vocab]``, caches ``[layers, slots, positions, kv_heads, dim]`` bf16, weights
``[layers, slots, kv_heads, positions]`` float32, states ``[slots, ...]``.
"""

from __future__ import annotations

import math
import zlib

import torch

own = False  # whether `run` calls the framework's operators or computes their plain form

VOCAB = 128256
MODELS = {"llama-1b": dict(heads=32, kv_heads=8, dim=64), "llama-8b": dict(heads=32, kv_heads=8, dim=128)}
LOGITS = {"bf16": torch.bfloat16, "f32": torch.float32}


# ---- cases --------------------------------------------------------------------------------- #
def listed() -> list[dict]:
    return [
        # one user, four beams: the smallest selection, where launches count
        dict(name="beam-chat", kind="beam", groups=1, beams=4, vocab=VOCAB, k=4, dtype="bf16", ended=False),
        # a full batch of 64 rows; twice the beams as candidates, some beams have ended
        dict(name="beam-batch-64", kind="beam", groups=8, beams=8, vocab=VOCAB, k=16, dtype="bf16", ended=True),
        # 32-bit logits of a layer-list model with a vocabulary of odd size
        dict(name="beam-f32-odd", kind="beam", groups=3, beams=5, vocab=32003, k=10, dtype="f32", ended=True),
        # four beams a hundred tokens behind their prompt
        dict(name="reorder-chat", kind="reorder", model="llama-1b", layers=16, groups=1, beams=4, first=501, rows=101),
        # eight users with eight beams each, long answers of different lengths; depth cut (a layer is what repeats)
        dict(name="reorder-batch-64", kind="reorder", model="llama-8b", layers=8, groups=8, beams=8, first=256, rows=1024),
        # recurrent states of a layer-list model: 32-bit matrices, moved whole
        dict(name="reorder-states", kind="reorder", model="", layers=10, groups=1, beams=6, first=0, rows=0),
        # one token's attention over a long document
        dict(name="weights-token", kind="weights", model="llama-1b", layers=1, sequences=1, queries=1, longest=65001),
        # the last tokens of a document's prompt: the usual window before an eviction
        dict(name="weights-window", kind="weights", model="llama-8b", layers=1, sequences=1, queries=64, longest=32768),
        # all queries of a prompt
        dict(name="weights-prompt", kind="weights", model="llama-1b", layers=1, sequences=1, queries=1501, longest=1501),
        # a short cache cut to a third
        dict(name="evict-short", kind="evict", model="llama-8b", layers=4, sequences=1, longest=1500, keep=512, sinks=4, recent=64),
        # several sequences of different lengths, some of them short enough to stay whole
        dict(name="evict-batch-7", kind="evict", model="llama-8b", layers=8, sequences=7, longest=4096, keep=1024, sinks=4, recent=128),
        # a long document's cache cut to an eighth, at full depth
        dict(name="evict-long", kind="evict", model="llama-1b", layers=16, sequences=1, longest=65001, keep=8192, sinks=4, recent=256),
    ]


def draw(rng) -> dict:
    def spread(low, high):
        return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))

    kind = rng.choice(["beam", "reorder", "weights", "evict"])
    model = rng.choice(sorted(MODELS))
    if kind == "beam":
        beams = rng.randint(1, 16)
        groups, vocab = spread(1, 64 // beams), spread(1000, VOCAB)
        return dict(kind=kind, groups=groups, beams=beams, vocab=vocab, k=beams * rng.choice([1, 2]), dtype=rng.choice(sorted(LOGITS)), ended=rng.random() < 0.5)
    if kind == "reorder":
        if rng.random() < 0.25:
            return dict(kind=kind, model="", layers=rng.randint(1, 16), groups=1, beams=rng.randint(2, 8), first=0, rows=0)
        beams = rng.randint(2, 8)
        return dict(kind=kind, model=model, layers=rng.randint(1, 8), groups=spread(1, 64 // beams), beams=beams, first=spread(1, 600), rows=spread(1, 1024))
    if kind == "weights":
        queries = spread(1, 1501)
        longest = max(queries, spread(64, min(65001, 2300000 // queries)))
        return dict(kind=kind, model=model, layers=1, sequences=1 if queries > 64 or longest > 8192 else rng.randint(1, 4), queries=queries, longest=longest)
    longest = spread(100, 32768)
    sinks, recent = rng.randint(0, 8), spread(1, 48)
    return dict(kind=kind, model=model, layers=rng.randint(1, 8), sequences=1 if longest > 8192 else rng.randint(1, 7), longest=longest,
                keep=max(64, spread(64, longest)), sinks=sinks, recent=recent)


# ---- inputs -------------------------------------------------------------------------------- #
def generator(seed: int, name: str) -> torch.Generator:
    return torch.Generator(device="cuda").manual_seed(zlib.crc32(f"{seed} {name}".encode()))


def normal(seed: int, name: str, shape, dtype=torch.bfloat16, std: float = 1.0) -> torch.Tensor:
    return torch.empty(shape, device="cuda", dtype=dtype).normal_(0.0, std, generator=generator(seed, name))


def whole(seed: int, name: str, low: int, high: int, shape) -> torch.Tensor:
    """int32 in [low, high)."""
    return torch.randint(low, high, shape, generator=generator(seed, name), device="cuda", dtype=torch.int32)


def cache_shape(case: dict, positions: int, slots: int):
    m = MODELS[case["model"]]
    return (case["layers"], slots, positions, m["kv_heads"], m["dim"])


def lengths_of(case: dict, seed: int) -> torch.Tensor:
    """The first sequence is the longest, the others are between a quarter of it and all of it."""
    n, b = case["longest"], case["sequences"]
    lengths = whole(seed, "lengths", max(n // 4, case.get("queries", 1)), n + 1, (b,))
    lengths[0] = n
    return lengths


def prepare(case: dict, seed: int) -> dict:
    kind, s = case["kind"], {"case": case}
    if kind == "beam":
        rows = case["groups"] * case["beams"]
        s["logits"] = normal(seed, "logits", (rows, case["vocab"]), LOGITS[case["dtype"]], 2.5)
        # (summed log-probabilities of a short answer)
        s["scores"] = normal(seed, "scores", (case["groups"], case["beams"]), torch.float32, 2.0) - 10
        ended = torch.rand(case["groups"], case["beams"], generator=generator(seed, "ended"), device="cuda") < 0.2
        s["done"] = ended.to(torch.uint8) if case["ended"] else None
        s["eos"] = case["vocab"] - 7
    elif kind == "reorder":
        slots = case["groups"] * case["beams"]
        group = torch.arange(slots, device="cuda", dtype=torch.int32) // case["beams"]
        s["parents"] = group * case["beams"] + whole(seed, "parents", 0, case["beams"], (slots,))
        if case["model"]:
            longest = case["first"] + case["rows"]
            # the beams of a group are equally long
            behind = whole(seed, "behind", (case["rows"] + 1) // 2, case["rows"] + 1, (case["groups"],))
            behind[0] = case["rows"]
            s["lengths"] = (case["first"] + behind).repeat_interleave(case["beams"])
            s["tensors"] = [normal(seed, n, cache_shape(case, longest + 11, slots)) for n in ("keys", "values")]
        else:
            s["lengths"] = None
            s["tensors"] = [normal(seed, f"state {i}", (slots, 32, 64, 64), torch.float32) for i in range(case["layers"])]
    elif kind == "weights":
        m, b = MODELS[case["model"]], case["sequences"]
        s["lengths"] = lengths_of(case, seed)
        s["q"] = normal(seed, "q", (case["layers"], b, case["queries"], m["heads"], m["dim"]))
        s["keys"] = normal(seed, "keys", cache_shape(case, case["longest"] + 5, b))
        s["weights"] = torch.zeros(case["layers"], b, m["kv_heads"], case["longest"] + 5, device="cuda")
    else:
        m, b = MODELS[case["model"]], case["sequences"]
        s["lengths"] = lengths_of(case, seed)
        shape = cache_shape(case, case["longest"] + 5, b)
        s["keys"], s["values"] = normal(seed, "keys", shape), normal(seed, "values", shape)
        # a few keys receive most of the weight; keys that nobody looked at have equal weights of zero
        w = normal(seed, "weights", (case["layers"], b, m["kv_heads"], case["longest"] + 5), torch.float32, 2.0).exp()
        s["weights"] = torch.where(w < 0.05, torch.zeros_like(w), w)
    return s


# ---- the operators' plain forms --------------------------------------------------------------- #
def plain_beam(s: dict):
    case, logits = s["case"], s["logits"].double()  # (neighbouring candidates decide which are taken)
    groups, beams, vocab, k = case["groups"], case["beams"], case["vocab"], case["k"]
    top = logits.max(dim=1, keepdim=True).values
    log_sum = (logits - top).exp().sum(dim=1, keepdim=True).log() + top
    score = s["scores"].double().reshape(-1, 1) + (logits - log_sum)
    if s["done"] is not None:
        end = torch.full_like(score, -math.inf)
        end[:, s["eos"]] = s["scores"].double().reshape(-1)
        score = torch.where(s["done"].reshape(-1, 1) != 0, end, score)
    best, at = torch.sort(score.view(groups, beams * vocab), dim=1, descending=True, stable=True)
    at, group = at[:, :k], torch.arange(groups, device=at.device).unsqueeze(1)
    parents, tokens = (at // vocab + group * beams).int(), (at % vocab).int()
    done = tokens == s["eos"]
    if s["done"] is not None:
        done = done | (s["done"].reshape(-1)[parents.long()] != 0)
    return best[:, :k].float(), parents, tokens, done.to(torch.uint8)


def plain_reorder(s: dict):
    case, parents = s["case"], s["parents"].long()
    if s["lengths"] is None:
        for t in s["tensors"]:
            t.copy_(t[parents])
        return s["tensors"]
    lo, hi = case["first"], case["first"] + case["rows"]
    row = torch.arange(lo, hi, device=parents.device)
    moves = (row[None, :] < s["lengths"].long()[parents][:, None])[None, :, :, None, None]
    for t in s["tensors"]:
        part = t[:, :, lo:hi]
        part.copy_(torch.where(moves, part[:, parents], part))
    return s["tensors"]


def plain_weights(s: dict):
    q, keys, weights = s["q"].float(), s["keys"].float(), s["weights"]
    layers, b, n, heads, dim = q.shape
    kv_heads, rows = keys.shape[3], keys.shape[2]
    q = q.view(layers, b, n, kv_heads, heads // kv_heads, dim).permute(0, 1, 3, 4, 2, 5).reshape(layers, b, kv_heads, -1, dim)
    scores = torch.matmul(q, keys.permute(0, 1, 3, 4, 2)).mul_(dim**-0.5)
    last = s["lengths"].view(b, 1) - n + torch.arange(n, device=q.device)  # the last row that a query sees
    hidden = torch.arange(rows, device=q.device) > last.repeat(1, heads // kv_heads).unsqueeze(-1)
    scores.masked_fill_(hidden[None, :, None], -math.inf)
    scores.sub_(scores.max(dim=-1, keepdim=True).values).exp_()
    scores.div_(scores.sum(dim=-1, keepdim=True))
    weights += scores.sum(dim=-2)
    return weights


def plain_evict(s: dict):
    case, weights, lengths = s["case"], s["weights"], s["lengths"].long()
    keep, rows = case["keep"], weights.shape[-1]
    row = torch.arange(rows, device=weights.device)
    held = (row < case["sinks"]) | (row >= lengths.view(-1, 1) - case["recent"])
    rank = torch.where(held[None, :, None], torch.full_like(weights, math.inf), weights)
    rank = torch.where((row >= lengths.view(-1, 1))[None, :, None], torch.full_like(weights, -math.inf), rank)
    taken = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :keep]
    count = lengths.clamp(max=keep)
    there = (torch.arange(keep, device=row.device) < count.view(-1, 1))[None, :, None]
    taken = torch.where(there, taken, torch.full_like(taken, rows)).sort(dim=-1).values
    taken = torch.where(there, taken, torch.full_like(taken, -1))
    source = taken.clamp(min=0).transpose(2, 3).unsqueeze(-1).expand(-1, -1, -1, -1, s["keys"].shape[-1])
    stays = there.transpose(2, 3).unsqueeze(-1)
    for t in (s["keys"], s["values"]):
        front = t[:, :, :keep]
        front.copy_(torch.where(stays, t.gather(2, source), front))
    return s["keys"], s["values"], taken.int()


# ---- one pass -------------------------------------------------------------------------------- #
def run(s: dict):
    kind = s["case"]["kind"]
    if not own:
        return {"beam": plain_beam, "reorder": plain_reorder, "weights": plain_weights, "evict": plain_evict}[kind](s)
    from megakernels_b200.native import mk_sequences as ops

    case = s["case"]
    if kind == "beam":
        return ops.beam_select(s["logits"], s["scores"], beams=case["beams"], k=case["k"], done=s["done"], eos=s["eos"])
    if kind == "reorder":
        if s["lengths"] is None:
            ops.reorder_slots(s["tensors"], s["parents"])
        else:
            ops.reorder_slots(s["tensors"], s["parents"], dim=1, first=case["first"], lengths=s["lengths"])
        return s["tensors"]
    if kind == "weights":
        ops.key_weights(s["q"], s["keys"], s["weights"], s["lengths"], scale=s["q"].shape[-1] ** -0.5)
        return s["weights"]
    rows = ops.select_rows(s["weights"], s["lengths"], keep=case["keep"], sinks=case["sinks"], recent=case["recent"])
    ops.move_rows(s["keys"], s["values"], rows, s["lengths"])
    return s["keys"], s["values"], rows


# ---- what a pass cannot do without -------------------------------------------------------------- #
def mean_length(case: dict) -> float:
    """Of the sequences that `lengths_of` makes."""
    n, b = case["longest"], case["sequences"]
    return (n + (b - 1) * (max(n // 4, case.get("queries", 1)) + n) / 2) / b


def work(case: dict) -> dict:
    kind = case["kind"]
    if kind == "beam":
        count = case["groups"] * case["beams"] * case["vocab"]
        return {"bytes": count * (2 if case["dtype"] == "bf16" else 4) + 13 * case["groups"] * case["k"], "flops": 3 * count}
    if kind == "reorder":
        b = case["beams"]
        moved, read = b - 1, b * (1 - (1 - 1 / b) ** (b - 1))  # parents are any of the group's
        if case["model"]:
            m = MODELS[case["model"]]
            rows = case["rows"] * (1 + (case["groups"] - 1) * 0.75) / case["groups"]
            slot = rows * case["layers"] * 2 * m["kv_heads"] * m["dim"] * 2
        else:
            slot = case["layers"] * 32 * 64 * 64 * 4
        return {"bytes": case["groups"] * (moved + read) * slot, "flops": 0}
    m = MODELS[case["model"]]
    items, length = case["layers"] * case["sequences"], mean_length(case)
    if kind == "weights":
        n = case["queries"]
        scores = n * (length - (n - 1) / 2) * m["heads"]
        moved = length * m["kv_heads"] * (m["dim"] * 2 + 8) + n * m["heads"] * m["dim"] * 2
        return {"bytes": items * moved, "flops": items * scores * (2 * m["dim"] + 4)}
    kept = min(case["keep"], length)
    return {"bytes": items * m["kv_heads"] * (4 * length + 4 * case["keep"] + kept * 2 * 2 * 2 * m["dim"]), "flops": items * m["kv_heads"] * length}


# ---- the same in 64 bits, from the definitions ------------------------------------------------- #
def exact(case: dict, seed: int):
    s = prepare(case, seed)
    if case["kind"] == "beam":
        p = torch.log_softmax(s["logits"].double(), dim=1).view(case["groups"], case["beams"], case["vocab"])
        total = p + s["scores"].double().unsqueeze(-1)
        if s["done"] is not None:
            over = s["done"] != 0
            total[over] = -math.inf
            total[..., s["eos"]] = torch.where(over, s["scores"].double(), total[..., s["eos"]])
        return total.flatten(1).topk(case["k"], dim=1).values, None, None, None
    if case["kind"] == "reorder":
        out = []
        for t in s["tensors"]:
            new = t.clone()
            for slot, parent in enumerate(s["parents"].tolist()):
                if s["lengths"] is None:
                    new[slot] = t[parent]
                else:
                    a, b = case["first"], int(s["lengths"][parent])
                    new[:, slot, a:b] = t[:, parent, a:b]
            out.append(new)
        return out
    if case["kind"] == "weights":
        m, n = MODELS[case["model"]], case["queries"]
        per = m["heads"] // m["kv_heads"]
        out = s["weights"].double()
        for layer in range(case["layers"]):
            for b, length in enumerate(s["lengths"].tolist()):
                seen = torch.arange(length, device="cuda")[None, :] <= torch.arange(length - n, length, device="cuda")[:, None]
                for h in range(m["heads"]):
                    z = s["q"][layer, b, :, h].double() @ s["keys"][layer, b, :length, h // per].double().T * m["dim"] ** -0.5
                    out[layer, b, h // per, :length] += torch.softmax(z.masked_fill(~seen, -math.inf), dim=-1).sum(dim=0)
        return out
    out = [s["keys"].clone(), s["values"].clone()]
    weights, rows = s["weights"].cpu().double(), s["weights"].shape[-1]
    place = torch.arange(rows)
    for layer in range(case["layers"]):
        for b, length in enumerate(s["lengths"].tolist()):
            for g in range(weights.shape[2]):
                w = weights[layer, b, g, :length].clone()
                w[: case["sinks"]] = math.inf
                w[max(0, length - case["recent"]):] = math.inf
                order = sorted(range(length), key=lambda j, w=w.tolist(): (-w[j], j))[: case["keep"]]
                at = place[sorted(order)].to("cuda")
                for new, old in zip(out, (s["keys"], s["values"])):
                    new[layer, b, : len(at), g] = old[layer, b, at, g]
    return out[0], out[1], None
