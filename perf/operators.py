"""What is measured of the operators behind several answers to one prompt: attention for a batch of sequences that share a
long prefix in the paged cache (`ops.attention_shared_prefix`), and the draw of a token with temperature, top-k, top-p and
min-p from given random numbers, with the token's log-probability (`ops.sample_filtered`).

Attention.  `groups` of sequences share the pages of their first positions; what follows is each sequence's own.  A page holds, a kv
head, the keys as [row][dim] and the values as [dim][row].  A step brings one token a sequence (decoding), or up to `new` of
them (questions behind one prompt, read in portions); a token at position p sees the keys 0 .. p.

The draw.  Tokens stand in descending order of their logits, ties by index, with weights exp((l - max) / T).  top_k keeps the
first k, top_p of those the shortest beginning that holds this share of their weight, min_p of those the ones with at
least that share of the largest weight; the token is the first at which the running sum of the kept weights passes u times
their sum.  A row with a temperature of 0 takes the first token.  The log-probability is that of softmax(logits) itself.
"""
import math
import random

import numpy as np
import torch

own = False

F32, F64 = torch.float32, torch.float64
TYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}


def _attention(name, dtype, heads, kv_heads, dim, requests, prefix, tail, new=1, groups=1, alone=0, page=16, softcap=0.0, sink=False, lengths=1):
    """requests sequences in `groups` groups behind prefixes of `prefix` positions (the first group's; the others' are shorter), with
    up to `tail` positions of their own each, and `alone` more that share nothing."""
    return {"name": name, "kind": "attention", "dtype": dtype, "heads": heads, "kv_heads": kv_heads, "dim": dim, "requests": requests,
            "prefix": prefix, "tail": tail, "new": new, "groups": groups, "alone": alone, "page": page, "softcap": softcap, "sink": sink,
            "lengths": lengths}


def _draws(name, rows, vocab, filters):
    return {"name": name, "kind": "sample", "rows": rows, "vocab": vocab, "filters": filters}


def listed():
    return [
        # four answers to a short prompt, the heads of the TinyLlama shape: launches and latency are all there is
        _attention("answers4_p300_h32x4d64_bf16", "bfloat16", 32, 4, 64, 4, 300, 40),
        # sixteen answers to an ordinary prompt
        _attention("answers16_p1500_h32x4d64_bf16", "bfloat16", 32, 4, 64, 16, 1500, 400, lengths=2),
        # the 32-bit path, a prompt whose last page is shared in part
        _attention("answers8_p1003_h32x4d64_fp32", "float32", 32, 4, 64, 8, 1003, 130, lengths=3),
        # a full batch behind a long system prompt, the heads of the Llama-3-8B shape
        _attention("batch64_p6000_h32x8d128_bf16", "bfloat16", 32, 8, 128, 64, 6000, 700, lengths=4),
        # three documents with several questions each, requests of no group beside them, capped scores and sinks, an odd head size
        _attention("docs3_p2500_h24x8d80_capped_bf16", "bfloat16", 24, 8, 80, 21, 2500, 250, groups=3, alone=3, page=32, softcap=30.0, sink=True,
                   lengths=5),
        # questions of some dozens of tokens each, read behind one document
        _attention("questions8_p4000_h32x8d128_bf16", "bfloat16", 32, 8, 128, 8, 4000, 90, new=90, lengths=6),
        # the longest: a batch behind a prefix of thirty thousand positions
        _attention("batch32_p30000_h32x8d128_bf16", "bfloat16", 32, 8, 128, 32, 30000, 300, lengths=7),
        # one answer's draw: latency
        _draws("draw1_v32000", 1, 32000, "all"),
        # a batch of the TinyLlama vocabulary, every row with its own filters
        _draws("draw64_v32000", 64, 32000, "all"),
        # an odd vocabulary and temperatures alone
        _draws("draw7_v50261_plain", 7, 50261, "none"),
        # a batch of the Llama-3-8B vocabulary with top-p alone
        _draws("draw64_v128256_top_p", 64, 128256, "top_p"),
        # the largest batch
        _draws("draw256_v128256", 256, 128256, "all"),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49)))))


def draw(rng):
    if rng.random() < 0.4:
        rows, vocab = _spread(rng, 1, 256), _spread(rng, 1000, 128256)
        case = _draws("", rows, vocab, rng.choice(["all", "all", "top_p", "none", "top_k"]))
    else:
        heads, kv_heads, dim = rng.choice([(32, 4, 64), (32, 8, 128), (24, 8, 80), (16, 16, 96), (8, 1, 128), (12, 4, 48), (4, 2, 16), (32, 32, 128), (8, 2, 256)])
        dtype = rng.choice(["bfloat16", "bfloat16", "float32"])
        requests, prefix = _spread(rng, 1, 64), _spread(rng, 16, 12000)
        new = _spread(rng, 2, 60) if rng.random() < 0.25 else 1
        if dtype == "float32":
            requests, prefix, new = min(requests, 16), min(prefix, 4000), min(new, 30)
        if new > 1:
            requests, prefix = min(requests, 8), min(prefix, 4000)
        if kv_heads > 8:
            requests, prefix = min(requests, 24), min(prefix, 6000)
        case = _attention("", dtype, heads, kv_heads, dim, requests, prefix, max(new, _spread(rng, 1, 500)), new=new,
                          groups=rng.choice([1, 1, 1, 2, 4]), alone=rng.choice([0, 0, 0, 1, 3]), page=rng.choice([16, 16, 32, 64]),
                          softcap=rng.choice([0.0, 0.0, 0.0, 20.0]), sink=rng.random() < 0.25, lengths=rng.randrange(1 << 30))
        case["groups"] = min(case["groups"], requests)
    del case["name"]
    return case


def _layout(case):
    """(first sequence, sequences, prefix) of the groups, and for every sequence its prefix, its length after the step and the
    tokens it brings in it."""
    rng = random.Random(case["lengths"])
    groups, sequences = [], []
    for index in range(case["groups"]):
        count = case["requests"] // case["groups"] + (1 if index < case["requests"] % case["groups"] else 0)
        prefix = max(1, case["prefix"] * (index + 2) // (2 * index + 2) - 3 * index)
        groups.append((len(sequences), count, prefix))
        for _ in range(count):
            new = rng.randint(1, case["new"])
            sequences.append((prefix, prefix + rng.randint(new, max(new, case["tail"])), new))
    for _ in range(case["alone"]):
        new = rng.randint(1, case["new"])
        sequences.append((0, rng.randint(new, max(new, case["tail"] + case["prefix"] // 4)), new))
    return groups, sequences


def prepare(case, seed):
    device = torch.device("cuda")
    gen = torch.Generator(device=device).manual_seed(seed)
    if case["kind"] == "sample":
        return _prepare_sample(case, seed, device, gen)
    groups, sequences = _layout(case)
    dtype, page, dim = TYPES[case["dtype"]], case["page"], case["dim"]
    # pages as the cache manager hands them out: in any order, those of a prefix once, in every row of its group
    blocks = max(length + page - 1 for _, length, _ in sequences) // page
    first_of = {first + i: first for first, count, _ in groups for i in range(count)}
    # (a page that a prefix fills in part is each sequence's own copy)
    shared = [prefix // page if first_of.get(row, row) != row else 0 for row, (prefix, _, _) in enumerate(sequences)]
    need = [(length + page - 1) // page for _, length, _ in sequences]
    total = sum(need) - sum(shared)
    order = np.random.RandomState(seed & 0x7fffffff).permutation(total)
    table, cursor = np.zeros((len(sequences), blocks), dtype=np.int32), 0
    for row in range(len(sequences)):
        fresh = need[row] - shared[row]
        table[row, :shared[row]] = table[first_of.get(row, row), :shared[row]]
        table[row, shared[row]:need[row]] = order[cursor:cursor + fresh]
        cursor += fresh
    cache = torch.randn((total, 2, case["kv_heads"], page * dim), device=device, generator=gen, dtype=F32).to(dtype)
    counts = np.array([new for _, _, new in sequences])
    seq_start = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    seq_len = np.array([length for _, length, _ in sequences], dtype=np.int32)
    # a sequence's own rows of a page that a prefix fills in part begin with a copy of the prefix's rows
    for first, count, prefix in groups:
        rest = prefix % page
        if rest:
            source, block = int(table[first, prefix // page]), prefix // page
            planes = cache.view(-1, 2, case["kv_heads"], page * dim)
            for row in range(first + 1, first + count):
                target = int(table[row, block])
                planes[target, 0, :, :rest * dim] = planes[source, 0, :, :rest * dim]
                planes[target, 1].view(-1, dim, page)[:, :, :rest] = planes[source, 1].view(-1, dim, page)[:, :, :rest]
    positions = np.concatenate([np.arange(length - new, length) for _, length, new in sequences]).astype(np.int32)
    # queries that look for something: scores with a deviation of about 1.5
    q = (1.5 * torch.randn((int(counts.sum()), case["heads"] * dim), device=device, generator=gen, dtype=F32)).to(dtype)
    state = {"kind": "attention", "q": q, "cache": cache, "table": torch.from_numpy(table).to(device), "positions": torch.from_numpy(positions).to(device),
             "seq_start": seq_start, "seq_len": seq_len, "groups": groups, "heads": case["heads"], "kv_heads": case["kv_heads"], "dim": dim,
             "page": page, "scale": 1.0 / math.sqrt(dim), "softcap": case["softcap"] or None,
             "sink": torch.randn((case["heads"],), device=device, generator=gen, dtype=F32) if case["sink"] else None, "sequences": sequences}
    if own:
        from tlie_amd import ops
        # a step's work list: made once, read by every layer of the step
        state["plan"] = ops.shared_prefix_plan(seq_start, seq_len, groups, case["heads"], case["kv_heads"], dim, dtype, device)
    return state


def _prepare_sample(case, seed, device, gen):
    rows, vocab = case["rows"], case["vocab"]
    # a model's logits: a broad bulk and a few tokens far above it, more or fewer of them from row to row
    logits = 2.0 * torch.randn((rows, vocab), device=device, generator=gen, dtype=F32)
    lifted = torch.rand((rows, vocab), device=device, generator=gen) < 40.0 / vocab
    logits += lifted * torch.rand((rows, vocab), device=device, generator=gen) * torch.linspace(4.0, 14.0, rows, device=device).unsqueeze(1)
    rng = random.Random(seed)
    filters = case["filters"]
    temperature = [rng.uniform(0.5, 1.3) for _ in range(rows)]
    top_k = [rng.choice([0, 20, 50, 400]) if filters in ("all", "top_k") else 0 for _ in range(rows)]
    top_p = [rng.choice([1.0, 0.95, 0.9, 0.6]) if filters in ("all", "top_p") else 1.0 for _ in range(rows)]
    min_p = [rng.choice([0.0, 0.02, 0.1]) if filters == "all" else 0.0 for _ in range(rows)]
    if filters == "all" and rows > 4:
        temperature[3] = 0.0
    tensor = lambda values, dtype: torch.tensor(values, dtype=dtype, device=device)
    return {"kind": "sample", "logits": logits, "uniform": torch.rand((rows,), device=device, generator=gen, dtype=F32),
            "temperature": tensor(temperature, F32), "top_k": tensor(top_k, torch.int32) if filters in ("all", "top_k") else None,
            "top_p": tensor(top_p, F32) if filters in ("all", "top_p") else None, "min_p": tensor(min_p, F32) if filters == "all" else None}


def run(state):
    if own:
        from tlie_amd import ops
        if state["kind"] == "sample":
            return ops.sample_filtered(state["logits"], state["uniform"], state["temperature"], top_k=state["top_k"], top_p=state["top_p"],
                                       min_p=state["min_p"], logprobs=True)
        return ops.attention_shared_prefix(state["q"], state["cache"], state["table"], state["positions"], state["plan"], state["heads"],
                                           state["kv_heads"], state["dim"], state["scale"], softcap=state["softcap"], sink=state["sink"])
    return _plain_sample(state) if state["kind"] == "sample" else _plain_attention(state)


def _keys_and_values(state, table):
    """The pages that `table` [..., blocks] names, as 32-bit keys and values [..., kv heads, positions, dim]."""
    page, dim, kv_heads = state["page"], state["dim"], state["kv_heads"]
    pages = state["cache"][table.long()].float()                                    # [..., blocks, 2, kv heads, page * dim]
    lead = pages.shape[:-4]
    count = pages.shape[-4] * page
    keys = pages[..., 0, :, :].unflatten(-1, (page, dim)).movedim(-3, -4).reshape(*lead, kv_heads, count, dim)
    values = pages[..., 1, :, :].unflatten(-1, (dim, page)).movedim(-3, -4).transpose(-1, -2).reshape(*lead, kv_heads, count, dim)
    return keys, values


def _plain_attention(state):
    heads, kv_heads, dim, page = state["heads"], state["kv_heads"], state["dim"], state["page"]
    per = heads // kv_heads
    q = state["q"]
    out = torch.empty_like(q)
    covered = {first + i for first, count, _ in state["groups"] for i in range(count)}
    sets = list(state["groups"]) + [(row, 1, 0) for row in range(len(state["seq_len"])) if row not in covered]
    start, lengths = state["seq_start"], state["seq_len"]

    def capped(scores):
        scores = scores * state["scale"]
        return state["softcap"] * torch.tanh(scores / state["softcap"]) if state["softcap"] else scores

    for first, count, prefix in sets:
        begin, end = int(start[first]), int(start[first + count])
        most = int(max(start[first + i + 1] - start[first + i] for i in range(count)))
        longest = int(max(lengths[first:first + count]))
        # the group's queries as [sequence, kv head, token of it and head of the kv head, dim], the shorter ones padded
        places = torch.full((count, most), end - begin, dtype=torch.long)
        for i in range(count):
            n = int(start[first + i + 1] - start[first + i])
            places[i, :n] = torch.arange(n) + int(start[first + i]) - begin
        places = places.to(q.device)
        mine = torch.cat([q[begin:end].float(), q.new_zeros((1, heads * dim), dtype=F32)])[places]
        mine = mine.view(count, most, kv_heads, per, dim).permute(0, 2, 1, 3, 4).reshape(count, kv_heads, most * per, dim)
        at = torch.cat([state["positions"][begin:end].long(), state["positions"].new_full((1,), longest - 1).long()])[places]
        # what follows the prefix, each sequence's own
        base = prefix // page
        keys, values = _keys_and_values(state, state["table"][first:first + count, base:(longest + page - 1) // page])
        scores = capped(mine @ keys.transpose(-1, -2)).view(count, kv_heads, most, per, -1)
        spot = base * page + torch.arange(keys.shape[-2], device=q.device)
        seen = (spot >= prefix) & (spot <= at.unsqueeze(-1))                          # [sequence, token, key]
        scores = scores.masked_fill(~seen[:, None, :, None, :], -math.inf)
        top = scores.amax(dim=-1)
        if prefix > 0:
            shared_keys, shared_values = _keys_and_values(state, state["table"][first, :(prefix + page - 1) // page])
            flat = mine.transpose(0, 1).reshape(kv_heads, count * most * per, dim)
            shared = capped(flat @ shared_keys[:, :prefix].transpose(-1, -2))
            back = lambda x: x.view(kv_heads, count, most, per, *x.shape[2:]).transpose(0, 1)
            top = torch.maximum(top, back(shared.amax(dim=-1)))
        if state["sink"] is not None:
            sink = state["sink"].view(1, kv_heads, 1, per)
            top = torch.maximum(top, sink)
        weights = torch.exp(scores - top.unsqueeze(-1))
        total = weights.sum(dim=-1)
        result = (weights.view(count, kv_heads, most * per, -1) @ values).view(count, kv_heads, most, per, dim)
        if prefix > 0:
            shared = torch.exp(shared - top.transpose(0, 1).reshape(kv_heads, -1, 1))
            total = total + back(shared.sum(dim=-1))
            result = result + back(shared @ shared_values[:, :prefix])
        if state["sink"] is not None:
            total = total + torch.exp(sink - top)
        result = (result / total.unsqueeze(-1)).permute(0, 2, 1, 3, 4).reshape(count * most, heads * dim)
        flat_places = places.view(-1)
        live = flat_places < end - begin
        out[begin + flat_places[live]] = result[live].to(q.dtype)
    return out


def _plain_sample(state):
    # (in 64 bits: the draw compares running sums with a number, and a sum next to it decides a token)
    logits = state["logits"]
    rows, vocab = logits.shape
    ordered, index = torch.sort(logits, dim=-1, descending=True, stable=True)
    gap = ordered.double() - ordered[:, :1].double()
    temperature = state["temperature"].double().unsqueeze(1)
    greedy = ~(temperature > 0)
    weights = torch.exp(gap / torch.where(greedy, torch.ones_like(temperature), temperature))
    place = torch.arange(vocab, device=logits.device).unsqueeze(0)
    kept = torch.ones_like(weights, dtype=torch.bool)
    if state["top_k"] is not None:
        top_k = state["top_k"].long().unsqueeze(1)
        kept &= (place < top_k) | (top_k <= 0)
    if state["top_p"] is not None:
        top_p = state["top_p"].double().unsqueeze(1)
        running = torch.cumsum(weights * kept, dim=-1)
        before = torch.cat([torch.zeros_like(running[:, :1]), running[:, :-1]], dim=-1)
        kept &= (before < top_p * running[:, -1:]) | ~(top_p < 1)
    if state["min_p"] is not None:
        kept &= weights >= state["min_p"].double().unsqueeze(1)
    kept[:, 0] = True
    running = torch.cumsum(weights * kept, dim=-1)
    goal = state["uniform"].double().unsqueeze(1) * running[:, -1:]
    chosen = (running <= goal).sum(dim=-1, keepdim=True)
    chosen = torch.minimum(chosen, kept.sum(dim=-1, keepdim=True) - 1)
    chosen = torch.where(greedy, torch.zeros_like(chosen), chosen)
    tokens = torch.gather(index, 1, chosen).squeeze(1).int()
    logprobs = torch.gather(gap, 1, chosen).squeeze(1) - torch.log(torch.exp(gap).sum(dim=-1))
    return tokens, logprobs.float()


def work(case):
    if case["kind"] == "sample":
        count = case["rows"] * case["vocab"]
        return {"bytes": 4 * count + 28 * case["rows"], "flops": 4 * count}        # a weight is a subtraction, a product, an exponential and a sum
    groups, sequences = _layout(case)
    size = 2 if case["dtype"] == "bfloat16" else 4
    keys = sum(prefix for _, _, prefix in groups) + sum(length - prefix for prefix, length, _ in sequences)
    tokens = sum(new for _, _, new in sequences)
    pairs = sum(sum(range(length - new + 1, length + 1)) for _, length, new in sequences)
    return {"bytes": size * (keys * 2 * case["kv_heads"] * case["dim"] + 2 * tokens * case["heads"] * case["dim"]),
            "flops": 4 * case["dim"] * case["heads"] * pairs}


def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] == "sample":
        return _exact_sample(state)
    heads, kv_heads, dim, page = state["heads"], state["kv_heads"], state["dim"], state["page"]
    per = heads // kv_heads
    out = torch.empty((state["q"].shape[0], heads * dim), dtype=F64, device=state["q"].device)
    token = 0
    for row, (_, length, new) in enumerate(state["sequences"]):
        spots = torch.arange(length, device=out.device)
        pages, rows = state["table"][row].long()[spots // page], spots % page
        planes = state["cache"].view(-1, 2, kv_heads, page * dim)
        keys = planes[:, 0].view(-1, kv_heads, page, dim)[pages, :, rows].to(F64).movedim(0, 1).contiguous()       # [kv head, position, dim]
        values = planes[:, 1].view(-1, kv_heads, dim, page)[pages, :, :, rows].to(F64).movedim(0, 1).contiguous()
        for first in range(0, new, 32):                                # (some tokens at a time: the scores of all would be many)
            count = min(32, new - first)
            ask = state["q"][token + first:token + first + count].to(F64).view(count, kv_heads, per, dim).movedim(0, 1).reshape(kv_heads, count * per, dim)
            scores = torch.matmul(ask, keys.transpose(1, 2)) * state["scale"]
            if state["softcap"]:
                scores = torch.tanh(scores / state["softcap"]) * state["softcap"]
            scores = scores.view(kv_heads, count, per, length)
            ahead = spots > (length - new + first + torch.arange(count, device=out.device)).unsqueeze(1)
            scores = scores.masked_fill(ahead.view(1, count, 1, length), -math.inf)
            if state["sink"] is not None:
                sink = state["sink"].to(F64).view(kv_heads, 1, per, 1).expand(kv_heads, count, per, 1)
                share = torch.softmax(torch.cat([scores, sink], dim=-1), dim=-1)[..., :length]
            else:
                share = torch.softmax(scores, dim=-1)
            got = torch.matmul(share.reshape(kv_heads, count * per, length), values).view(kv_heads, count, per, dim)
            out[token + first:token + first + count] = got.movedim(0, 1).reshape(count, heads * dim)
        token += new
    return out


def _exact_sample(state):
    logits = state["logits"].cpu().numpy()
    host = {name: value.tolist() for name, value in state.items() if isinstance(value, torch.Tensor) and name != "logits"}
    number = lambda name, row: host[name][row] if name in host else None
    tokens, logprobs = [], []
    for row in range(logits.shape[0]):
        values = logits[row].astype(np.float64)
        order = np.lexsort((np.arange(values.size), -values))
        gap = values[order] - values[order[0]]
        temperature = number("temperature", row)
        if temperature > 0:
            weights = np.exp(gap / temperature)
            kept = values.size
            if number("top_k", row):
                kept = min(kept, int(number("top_k", row)))
            if number("top_p", row) is not None and number("top_p", row) < 1.0:
                sums = np.cumsum(weights[:kept])
                kept = min(kept, int(np.searchsorted(sums, number("top_p", row) * sums[-1], side="left")) + 1)
            if number("min_p", row):
                kept = max(1, int(np.count_nonzero(weights[:kept] >= number("min_p", row))))
            sums = np.cumsum(weights[:kept])
            pick = min(kept - 1, int(np.searchsorted(sums, number("uniform", row) * sums[-1], side="right")))
        else:
            pick = 0
        tokens.append(int(order[pick]))
        logprobs.append(gap[pick] - math.log(np.exp(gap).sum()))
    return np.array(tokens, dtype=np.int32), np.array(logprobs)
