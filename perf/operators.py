"""The operators of a beam search step, as cases to measure: selection over beams and vocabulary,
reordering of the survivors' states, and the sequences out of the recorded choices.

`run` computes a case in its plain form (elementary torch operations) or, where `own` is true, through
the library's entry points (radx_amd.BeamSelector, radx_amd.beam_reorder, radx_amd.beam_backtrace).
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}

SELECT_MOST = 64 * 8 * 131072 * 2   # bytes of the largest selection's logits
REORDER_MOST = 2 * 10 ** 9          # bytes of the largest call's states
BACKTRACE_MOST = 4096 * 64 * 8      # recorded places


def _select(name, batch, beams, vocab, k, dtype, pad=0, allowed=1.0, shared=False, finished=0.0, normalize=True):
    """pad: columns behind the vocabulary; allowed: share of the tokens that the mask leaves (1: no mask),
    one mask for all rows where `shared`; finished: share of the beams that have ended."""
    return {"name": name, "op": "select", "batch": batch, "beams": beams, "vocab": vocab, "k": k, "dtype": dtype, "pad": pad,
            "allowed": allowed, "shared": shared, "finished": finished, "normalize": normalize}


def _reorder(name, batch, beams, states, heads, positions, width, dtype, in_place=True, length=1.0, ragged=False):
    """states: tensors [batch * beams, heads, positions, width]; length: share of the positions in use;
    ragged: each batch item has a length of its own, handed over as a tensor."""
    return {"name": name, "op": "reorder", "batch": batch, "beams": beams, "states": states, "heads": heads, "positions": positions,
            "width": width, "dtype": dtype, "in_place": in_place, "length": length, "ragged": ragged}


def _backtrace(name, steps, batch, beams, ragged=False):
    return {"name": name, "op": "backtrace", "steps": steps, "batch": batch, "beams": beams, "ragged": ragged}


def listed():
    return [
        # one request, four beams, twice as many candidates as beams: the smallest step of an interactive server
        _select("select one request", 1, 4, 32000, 8, "f32"),
        # a small batch over an odd vocabulary whose rows are padded to a round length by the output layer
        _select("select odd vocabulary", 8, 5, 50001, 10, "bf16", pad=47),
        # decoding under a grammar: a mask for each beam, an eighth of the beams finished
        _select("select under masks", 16, 8, 65536, 16, "f16", allowed=0.05, finished=0.125),
        # log probabilities from elsewhere (several models' mean): no normalisation, float32
        _select("select log probabilities", 32, 6, 40000, 12, "f32", normalize=False),
        # a wide search: many beams, many candidates
        _select("select wide beams", 4, 32, 100003, 64, "bf16"),
        # offline decoding at the largest batch
        _select("select large batch", 64, 8, 131072, 16, "bf16"),
        # one request's short cache: latency
        _reorder("reorder one request", 1, 4, 8, 8, 256, 128, "bf16", length=0.3),
        # an ordinary batch with sequences of different lengths in a padded cache
        _reorder("reorder ragged batch", 16, 5, 8, 8, 1024, 128, "bf16", ragged=True),
        # the largest cache, in place
        _reorder("reorder long cache", 16, 8, 8, 8, 900, 128, "f16"),
        # recurrent states of odd width into a second set of buffers
        _reorder("reorder recurrent states", 24, 6, 4, 1, 16, 4101, "f32", in_place=False),
        # the sequences of one short answer, and of a large batch of long ones
        _backtrace("backtrace short", 200, 1, 4),
        _backtrace("backtrace long", 4096, 64, 8, ragged=True),
    ]


def _between(rng, low, high):
    """A whole number between low and high, spread over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.999)))))))


def draw(rng):
    op = rng.choice(["select", "select", "reorder", "backtrace"])
    if op == "select":
        batch, beams = _between(rng, 1, 64), _between(rng, 1, 32)
        dtype = rng.choice(["f32", "bf16", "bf16", "f16"])
        vocab = _between(rng, 2000, min(160000, SELECT_MOST // (batch * beams * (4 if dtype == "f32" else 2))))
        k = min(64, rng.choice([beams, 2 * beams, 2 * beams, _between(rng, 1, 64)]))
        return _strip(_select("", batch, beams, vocab, k, dtype, pad=rng.choice([0, 0, -vocab % 64, rng.randint(1, 99)]),
                              allowed=rng.choice([1.0, 1.0, 0.5, 0.02]), shared=rng.random() < 0.3, finished=rng.choice([0.0, 0.0, 0.2]),
                              normalize=rng.random() < 0.8))
    if op == "reorder":
        batch, beams, states = _between(rng, 1, 32), _between(rng, 2, 16), _between(rng, 1, 12)
        dtype = rng.choice(["bf16", "f16", "f32"])
        row = REORDER_MOST // (2 * batch * beams * states * (4 if dtype == "f32" else 2))
        heads = _between(rng, 1, 16)
        width = _between(rng, 1, min(600, max(1, row // heads)))
        positions = _between(rng, 1, max(1, min(4096, row // (heads * width))))
        in_place = rng.random() < 0.7
        return _strip(_reorder("", batch, beams, states, heads, positions, width, dtype, in_place=in_place,
                               length=rng.choice([1.0, rng.random()]), ragged=in_place and rng.random() < 0.4))
    batch, beams = _between(rng, 1, 64), _between(rng, 1, 32)
    return _strip(_backtrace("", _between(rng, 1, min(8192, BACKTRACE_MOST // (batch * beams))), batch, beams, ragged=rng.random() < 0.5))


def _strip(case):
    del case["name"]
    return case


def _positions(case):
    """The positions in use where all batch items have the same."""
    return max(1, min(case["positions"], int(round(case["positions"] * case["length"]))))


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))

    def whole(low, high, shape):
        return torch.randint(low, high, shape, generator=g, device="cuda", dtype=torch.int32)

    if case["op"] == "select":
        batch, beams, vocab = case["batch"], case["beams"], case["vocab"]
        rows = batch * beams
        # logits as an output layer leaves them: a bell with a spread of a few units, and rows that differ in it
        spread = torch.rand(rows, 1, generator=g, device="cuda") * 2.0 + 1.5
        logits = torch.randn(rows, vocab + case["pad"], generator=g, device="cuda").mul_(spread)
        if not case["normalize"]:
            logits = torch.log_softmax(logits[:, :vocab], 1)
        if case["pad"] and case["normalize"]:
            logits[:, vocab:] = 1000.0  # nothing of the padding belongs to the row
        cum = -torch.rand(batch, beams, generator=g, device="cuda") * 4.0 - 5.0
        allowed = finished = None
        if case["allowed"] < 1.0:
            some = 1 if case["shared"] else rows
            bits = (torch.rand(some, (vocab + 31) // 32, 32, generator=g, device="cuda") < case["allowed"]).to(torch.int64)
            words = (bits << torch.arange(32, device="cuda")).sum(2)
            allowed = torch.where(words >= 1 << 31, words - (1 << 32), words).to(torch.int32)
        if case["finished"]:
            finished = torch.rand(batch, beams, generator=g, device="cuda") < case["finished"]
        state = {"logits": logits.to(DTYPES[case["dtype"]])[:, :vocab], "cum": cum, "allowed": allowed, "finished": finished,
                 "end": 2 if finished is not None else None}
        if own:
            import radx_amd
            state["selector"] = radx_amd.BeamSelector(batch, beams, vocab, case["k"])
    elif case["op"] == "reorder":
        batch, beams = case["batch"], case["beams"]
        shape = (batch * beams, case["heads"], case["positions"], case["width"])
        lengths = whole(1, case["positions"] + 1, (batch,)) if case["ragged"] else None
        states = [torch.randn(shape, generator=g, device="cuda", dtype=DTYPES[case["dtype"]]) for _ in range(case["states"])]
        state = {"parents": whole(0, beams, (batch, beams)), "lengths": lengths, "states": states, "into": None}
        if not case["in_place"]:
            state["into"] = [torch.zeros_like(s) for s in states]
    else:
        shape = (case["steps"], case["batch"], case["beams"])
        state = {"tokens": whole(0, 100000, shape), "parents": whole(0, case["beams"], shape), "steps": None,
                 "out": torch.full((case["batch"], case["beams"], case["steps"]), -1, device="cuda", dtype=torch.int32)}
        if case["ragged"]:
            state["steps"] = whole((case["steps"] + 1) // 2, case["steps"] + 1, (case["batch"],))
    state["case"] = case
    return state


def run(state):
    case = state["case"]
    if case["op"] == "select":
        return _own_select(state, case) if own else _plain_select(state, case)
    if case["op"] == "reorder":
        return _own_reorder(state, case) if own else _plain_reorder(state, case)
    return _own_backtrace(state, case) if own else _plain_backtrace(state, case)


def _own_select(state, case):
    return state["selector"].select(state["logits"], state["cum"], case["k"], allowed=state["allowed"], finished=state["finished"],
                                    end_token=state["end"], normalize=case["normalize"])


def _own_reorder(state, case):
    import radx_amd
    if state["lengths"] is not None:
        radx_amd.beam_reorder(state["states"], state["parents"], lengths=state["lengths"], length_dim=2)
        return state["states"]
    used = [s[:, :, :_positions(case)] for s in state["states"]]
    if state["into"] is None:
        radx_amd.beam_reorder(used, state["parents"])
        return state["states"]
    radx_amd.beam_reorder(used, state["parents"], into=[s[:, :, :_positions(case)] for s in state["into"]])
    return state["into"]


def _own_backtrace(state, case):
    import radx_amd
    return radx_amd.beam_backtrace(state["tokens"], state["parents"], steps=state["steps"], out=state["out"])


def _plain_select(state, case):
    """In 64 bits: the order of two candidates hangs on the last digits of their rows' sums."""
    batch, beams, vocab, k = case["batch"], case["beams"], case["vocab"], case["k"]
    low = float("-inf")
    x = state["logits"].double()
    if state["allowed"] is not None:
        token = torch.arange(vocab, device=x.device)
        bit = (state["allowed"][:, token >> 5] >> (token & 31).to(torch.int32)) & 1
        x = torch.where(bit.bool(), x, low)
    top = x.amax(1, keepdim=True)
    log_sum = (x - top).exp().sum(1, keepdim=True).log()
    cum = state["cum"].double().reshape(-1, 1)
    fine = torch.isfinite(top) & torch.isfinite(log_sum) & torch.isfinite(cum)
    score = torch.where(fine, cum + ((x - top) - log_sum if case["normalize"] else x), low)
    if state["finished"] is not None:
        ended = state["finished"].reshape(-1, 1)
        score = torch.where(ended, low, score)
        score[:, state["end"]] = torch.where(ended, cum, score[:, state["end"]:state["end"] + 1])[:, 0]
    score = score.reshape(batch, beams * vocab)
    # the k largest values are certain whatever their places; of those equal to the last the lowest places are wanted
    most = min(k, beams * vocab)
    best, at = score.topk(most, 1)
    last = best[:, -1:]
    places = torch.arange(beams * vocab, device=x.device)
    far = beams * vocab
    tied = torch.where(score == last, places, far).topk(most, 1, largest=False).values
    value = torch.cat([torch.where(best > last, best, low), torch.where(tied < far, last, low)], 1)
    place = torch.cat([torch.where(best > last, at, far), tied], 1)
    place, order = place.sort(1)
    value, again = value.gather(1, order).sort(dim=1, descending=True, stable=True)
    place = place.gather(1, again)[:, :k]
    value = value[:, :k]
    none = value == low
    parents = torch.where(none, -1, place // vocab).to(torch.int32)
    tokens = torch.where(none, -1, place % vocab).to(torch.int32)
    if most < k:
        value = torch.nn.functional.pad(value, (0, k - most), value=low)
        parents = torch.nn.functional.pad(parents, (0, k - most), value=-1)
        tokens = torch.nn.functional.pad(tokens, (0, k - most), value=-1)
    if state["finished"] is None:
        return value.float(), parents, tokens
    ended = state["finished"].gather(1, parents.clamp(min=0).long()) | (tokens == state["end"])
    return value.float(), parents, tokens, ended & (parents >= 0)


def _plain_reorder(state, case):
    batch, beams = case["batch"], case["beams"]
    rows = (torch.arange(batch, device="cuda").reshape(-1, 1) * beams + state["parents"]).reshape(-1)
    if state["lengths"] is not None:
        position = torch.arange(case["positions"], device="cuda").reshape(1, 1, -1, 1)
        used = position < state["lengths"].repeat_interleave(beams).reshape(-1, 1, 1, 1)
        moved = [s.copy_(torch.where(used, s[rows], s)) for s in state["states"]]
        return moved
    n = _positions(case)
    into = state["states"] if state["into"] is None else state["into"]
    [d[:, :, :n].copy_(s[:, :, :n][rows]) for s, d in zip(state["states"], into)]
    return into


def _plain_backtrace(state, case):
    """The maps from a later step's places to an earlier one's, joined in doubling strides."""
    steps, batch, beams = case["steps"], case["batch"], case["beams"]
    step = torch.arange(steps, device="cuda").reshape(-1, 1, 1)
    ends = state["steps"].reshape(1, -1, 1) if state["steps"] is not None else torch.full((1, 1, 1), steps, device="cuda")
    itself = torch.arange(beams, device="cuda").expand(steps, batch, beams)
    back = torch.cat([state["parents"][1:].long(), itself[:1]])
    place = torch.where(step < ends - 1, back, itself)
    stride = 1
    while stride < steps:
        place = torch.cat([place[:-stride].gather(2, place[stride:]), place[-stride:]])
        stride *= 2
    found = state["tokens"].gather(2, place).permute(1, 2, 0)
    return torch.where((step < ends).permute(1, 2, 0), found, state["out"])


def work(case):
    if case["op"] == "select":
        rows = case["batch"] * case["beams"]
        live = rows * (1.0 - case["finished"])
        size = 4 if case["dtype"] == "f32" else 2
        masks = 0.0 if case["allowed"] >= 1.0 else (1 if case["shared"] else live) * ((case["vocab"] + 31) // 32) * 4
        out = case["batch"] * case["k"] * (13 if case["finished"] else 12)
        elements = live * case["vocab"] * (case["allowed"] if case["allowed"] < 1.0 else 1.0)
        # an element: difference, exponential, sum, and two comparisons (the maximum, the k-th best so far)
        return {"bytes": live * case["vocab"] * size + masks + rows * 4 + out, "flops": 5 * elements}
    if case["op"] == "reorder":
        b = case["beams"]
        share = 0.5 * (1 + 1 / case["positions"]) if case["ragged"] else _positions(case) / case["positions"]
        row = case["heads"] * case["positions"] * case["width"] * (4 if case["dtype"] == "f32" else 2) * share
        # parents are drawn evenly: the expected numbers of rows that go somewhere, and of rows that change
        read = b * (1 - (1 - 1 / b) ** (b - 1 if case["in_place"] else b))
        written = b - 1 if case["in_place"] else b
        return {"bytes": case["batch"] * case["states"] * row * (read + written) + case["batch"] * b * 4, "flops": 0}
    places = case["steps"] * case["batch"] * case["beams"]
    return {"bytes": places * (0.75 if case["ragged"] else 1.0) * 12, "flops": 0}


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "select":
        return _exact_select(state, case)
    if case["op"] == "reorder":
        return None  # the values that move are the values that were there
    tokens, parents = state["tokens"].cpu().numpy(), state["parents"].cpu().numpy()
    out = state["out"].cpu().numpy().copy()
    ends = np.full(case["batch"], case["steps"]) if state["steps"] is None else state["steps"].cpu().numpy()
    items = np.arange(case["batch"])[:, None]
    place = np.broadcast_to(np.arange(case["beams"]), (case["batch"], case["beams"])).copy()
    for t in range(case["steps"] - 1, -1, -1):
        live = t < ends
        out[live, :, t] = tokens[t][items, place][live]
        place[live] = parents[t][items, place][live]
    return out


def _exact_select(state, case):
    vocab, beams, k = case["vocab"], case["beams"], case["k"]
    cum = state["cum"].cpu().numpy().astype(np.float64)
    ended = state["finished"].cpu().numpy() if state["finished"] is not None else np.zeros(cum.shape, bool)
    words = state["allowed"].cpu().numpy().view(np.uint32) if state["allowed"] is not None else None
    scores = np.full((case["batch"], k), -np.inf)
    parents = np.full((case["batch"], k), -1, np.int32)
    tokens = np.full((case["batch"], k), -1, np.int32)
    flags = np.zeros((case["batch"], k), bool)
    for b in range(case["batch"]):
        x = state["logits"][b * beams:(b + 1) * beams].double().cpu().numpy()
        found = []
        for i in range(beams):
            if ended[b, i]:
                found.append((np.array([cum[b, i]]), np.array([i]), np.array([state["end"]])))
                continue
            ids = np.arange(vocab)
            if words is not None:
                row = words[0 if len(words) == 1 else b * beams + i]
                ids = np.flatnonzero(np.unpackbits(row.view(np.uint8), bitorder="little")[:vocab])
            if not len(ids):
                continue
            v = x[i, ids]
            s = v + cum[b, i]
            if case["normalize"]:
                s = s - np.logaddexp.reduce(v) if len(v) < 64 else s - (v.max() + np.log(math.fsum(np.exp(v - v.max()))))
            keep = np.arange(len(s))
            if len(s) > k:
                keep = np.flatnonzero(s >= np.partition(s, len(s) - k)[len(s) - k])
            found.append((s[keep], np.full(len(keep), i), ids[keep]))
        if not found:
            continue
        s, i, v = (np.concatenate(part) for part in zip(*found))
        order = np.lexsort((v, i, -s))[:k]
        scores[b, :len(order)], parents[b, :len(order)], tokens[b, :len(order)] = s[order], i[order], v[order]
        flags[b, :len(order)] = ended[b, i[order]] | (v[order] == state["end"])
    if state["finished"] is None:
        return scores, parents, tokens
    return scores, parents, tokens, flags
