"""Attention for sequences that share their first positions, against its definition in 64 bits.

Tolerances, with A = sum_j p_j |v_j| of the oracle: the probabilities of the bfloat16 kernel are rounded to bfloat16 (2^-8 of
each, at worst 2^-8 A) and so is the result (2^-8 |out|).  A score is a sum of d products in 32 bits, off by at most (d + 4) 2^-24 of
S = scale * sum |q| |k|; that moves a probability and the sum of all by that share each, 2 (d + 4) 2^-24 S A (a capped score by no more); sums
over n keys and exponentials add (n + 64) 2^-24 A."""
import math

import numpy as np
import pytest
import torch

from tlie_amd import ops
from tlie_amd.errors import EngineError

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(autouse=True, params=["as it comes", "cut into parts"])
def form(request, monkeypatch):
    """Short steps run in one launch; every step also runs cut into parts."""
    if request.param == "cut into parts":
        monkeypatch.setattr(ops, "direct_prefix_items", lambda *step: None)


def make_step(seed, dtype, heads, kv_heads, dim, page, sequences, groups, fill=1.0):
    """sequences: (length after the step, tokens it brings).  Sequences of a group have the pages of whole blocks of their prefix in
    common, and a copy of the prefix's rows on the page where it ends."""
    gen = torch.Generator().manual_seed(seed)
    need = [(length + page - 1) // page for length, _ in sequences]
    blocks = max(need) + 1
    order = torch.randperm(sum(need) + 5, generator=gen).tolist()
    pages = len(order)
    table = np.zeros((len(sequences), blocks), dtype=np.int32)
    for row in range(len(sequences)):
        table[row, :need[row]] = [order.pop() for _ in range(need[row])]
    cache = (torch.randn((pages, 2, kv_heads, page * dim), generator=gen) * fill).to(dtype)
    keys, values = cache[:, 0].view(pages, kv_heads, page, dim), cache[:, 1].view(pages, kv_heads, dim, page)
    for first, count, prefix in groups:
        for row in range(first + 1, first + count):
            table[row, :prefix // page] = table[first, :prefix // page]
            rest = prefix % page
            if rest:
                source, target = int(table[first, prefix // page]), int(table[row, prefix // page])
                keys[target, :, :rest], values[target, :, :, :rest] = keys[source, :, :rest], values[source, :, :, :rest]
    counts = [new for _, new in sequences]
    start = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    lengths = np.array([length for length, _ in sequences], dtype=np.int32)
    positions = np.concatenate([np.arange(length - new, length) for length, new in sequences]).astype(np.int32)
    q = (1.5 * torch.randn((int(start[-1]), heads * dim), generator=gen)).to(dtype)
    return dict(q=q, cache=cache, table=torch.from_numpy(table), start=start, lengths=lengths, positions=torch.from_numpy(positions), groups=groups,
                heads=heads, kv_heads=kv_heads, dim=dim, page=page, scale=1.0 / math.sqrt(dim), dtype=dtype)


def oracle(step, softcap=None, sink=None):
    """(out, bound on the kernel's error), float64."""
    heads, kv_heads, dim, page = step["heads"], step["kv_heads"], step["dim"], step["page"]
    out, bound = [], []
    half = 2.0 ** -8 if step["dtype"] == BF16 else 0.0
    for row, length in enumerate(step["lengths"].tolist()):
        spots = torch.arange(length)
        pages = step["table"][row].long()[spots // page]
        k = step["cache"][:, 0].view(-1, kv_heads, page, dim)[pages, :, spots % page].double()          # [length, kv heads, dim]
        v = step["cache"][:, 1].view(-1, kv_heads, dim, page)[pages, :, :, spots % page].double()
        for token in range(int(step["start"][row]), int(step["start"][row + 1])):
            seen = int(step["positions"][token]) + 1
            q = step["q"][token].double().view(heads, dim)
            for head in range(heads):
                kv = head // (heads // kv_heads)
                s = (k[:seen, kv] @ q[head]) * step["scale"]
                size = float((k[:seen, kv].abs() @ q[head].abs()).max()) * step["scale"]
                s = softcap * torch.tanh(s / softcap) if softcap else s
                top = max(float(s.max()), float(sink[head]) if sink is not None else -math.inf)
                p = torch.exp(s - top)
                p = p / (p.sum() + (math.exp(float(sink[head]) - top) if sink is not None else 0.0))
                result, spread = p @ v[:seen, kv], p @ v[:seen, kv].abs()
                out.append(result)
                bound.append(half * spread + half * result.abs() + (2 * (dim + 4) * size + seen + 64) * 2.0 ** -24 * spread)
    shape = (step["q"].shape[0], heads * dim)
    return torch.stack(out).reshape(shape), torch.stack(bound).reshape(shape)


def call(step, softcap=None, sink=None, plan=None):
    on = lambda name: step[name].to(DEV)
    plan = plan or ops.shared_prefix_plan(step["start"], step["lengths"], step["groups"], step["heads"], step["kv_heads"], step["dim"], step["dtype"], DEV)
    return ops.attention_shared_prefix(on("q"), on("cache"), on("table"), on("positions"), plan, step["heads"], step["kv_heads"], step["dim"],
                                       step["scale"], softcap=softcap, sink=sink.to(DEV) if sink is not None else None)


def check(step, softcap=None, sink=None):
    got = call(step, softcap, sink)
    want, bound = oracle(step, softcap, sink)
    assert got.dtype == step["dtype"]
    excess = (got.double().cpu() - want).abs() - bound
    assert float(excess.max()) <= 0.0, float(excess.max())
    return got


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("heads,kv_heads,dim,page", [(4, 2, 16, 16), (8, 1, 64, 16), (6, 2, 48, 32), (4, 4, 80, 16), (16, 2, 128, 64), (20, 1, 96, 16),
                                                     (2, 2, 112, 32), (4, 1, 144, 16), (4, 1, 256, 16)])
def test_decode_step(dtype, heads, kv_heads, dim, page):
    """Five answers behind a prefix that ends inside a page, and one request that shares nothing."""
    check(make_step(1, dtype, heads, kv_heads, dim, page, [(170, 1), (171, 1), (200, 1), (229, 1), (300, 1), (37, 1)], [(0, 5, 169)]))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("prefix", [1, 15, 16, 17, 31, 32, 33, 127, 128, 129, 640])
def test_where_the_prefix_ends(dtype, prefix):
    check(make_step(2, dtype, 8, 2, 64, 16, [(prefix + 1, 1), (prefix + 2, 1), (prefix + 40, 1)], [(0, 3, prefix)]))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 2, 64), (24, 8, 80), (40, 2, 32)])
def test_portions(dtype, heads, kv_heads, dim):
    """Several tokens a sequence, one sequence that brings none, groups in no order, a group of one, a prefix of nothing."""
    sequences = [(90, 20), (75, 5), (73, 3), (50, 0), (260, 33), (213, 1), (9, 9), (140, 2), (30, 7)]
    check(make_step(3, dtype, heads, kv_heads, dim, 16, sequences, [(4, 2, 212), (0, 3, 70), (7, 1, 100), (8, 1, 0)]))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_many_columns(dtype):
    """More tokens than one tile of columns holds, and parts of a long prefix."""
    check(make_step(4, dtype, 8, 2, 64, 16, [(1500 + 3 * i, 1) for i in range(1, 30)], [(0, 29, 1499)]))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("softcap,with_sink", [(20.0, False), (None, True), (5.0, True)])
def test_caps_and_sinks(dtype, softcap, with_sink):
    step = make_step(5, dtype, 8, 4, 64, 16, [(300, 1), (310, 4), (333, 1)], [(0, 2, 290)])
    sink = torch.linspace(-3.0, 6.0, 8) if with_sink else None
    got = check(step, softcap, sink)
    assert not torch.equal(got, call(step))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_a_long_sequence_of_its_own(dtype):
    """Own keys cut into parts, some of which only the later tokens see."""
    check(make_step(6, dtype, 4, 1, 64, 16, [(2300, 1), (2600, 600)], [(1, 1, 5)]) if dtype == BF16
          else make_step(6, dtype, 4, 1, 32, 16, [(2300, 1), (900, 300)], [(1, 1, 5)]))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_rows_nobody_wrote_reach_nothing(dtype):
    """NaN and infinities on the free pages, behind every sequence's end, and in the shared rows of pages that are not the first's."""
    step = make_step(7, dtype, 8, 2, 64, 16, [(75, 1), (92, 3), (100, 1), (20, 1)], [(0, 3, 70)])
    want, bound = oracle(step)
    page = step["page"]
    keys, values = step["cache"][:, 0].view(-1, 2, page, 64), step["cache"][:, 1].view(-1, 2, 64, page)
    live = torch.zeros((step["cache"].shape[0], page), dtype=torch.bool)
    for row, length in enumerate(step["lengths"].tolist()):
        for spot in range(length):
            if row in (1, 2) and spot < 70:
                continue                                  # read through the group's first sequence
            live[int(step["table"][row, spot // page]), spot % page] = True
    keys[(~live)[:, None, :].expand(-1, 2, -1)] = math.nan
    values.transpose(2, 3)[(~live)[:, None, :].expand(-1, 2, -1)] = math.inf
    excess = (call(step).double().cpu() - want).abs() - bound
    assert float(excess.max()) <= 0.0


def test_the_same_as_the_attention_that_reads_everything():
    """Two kernels for one definition: their results differ by both bounds at most, and by nothing from call to call."""
    step = make_step(8, BF16, 32, 4, 64, 16, [(700 + i, 1) for i in range(6)], [(0, 6, 690)])
    got = call(step)
    assert torch.equal(got, call(step))
    on = lambda name: step[name].to(DEV)
    other = ops.attention_mfma(on("q"), on("cache"), on("table"), None, on("positions"), 32, 4, 64, None, step["scale"])
    _, bound = oracle(step)
    assert float(((got.double() - other.double()).cpu().abs() - 2 * bound).max()) <= 0.0


def test_rows_of_no_sequence_are_zeros_and_empty_steps_are_steps():
    step = make_step(9, BF16, 4, 2, 32, 16, [(40, 1), (33, 1)], [(0, 2, 32)])
    plan = ops.shared_prefix_plan(step["start"], step["lengths"], step["groups"], 4, 2, 32, BF16, DEV)
    plan.part_first = torch.cat([plan.part_first, plan.part_first[-1:]])           # a padding token behind the last
    plan.tokens += 1
    step["q"] = torch.cat([step["q"], torch.full_like(step["q"][:1], math.nan)])
    step["positions"] = torch.cat([step["positions"], torch.zeros(1, dtype=torch.int32)])
    assert (call(step, plan=plan)[2] == 0).all()
    empty = make_step(9, BF16, 4, 2, 32, 16, [(40, 0)], [])
    assert call(empty).shape == (0, 128)


def test_another_stream_and_a_replayed_recording():
    step = make_step(10, BF16, 8, 2, 64, 16, [(500, 1), (480, 1), (476, 1)], [(0, 3, 470)])
    want = call(step)
    plan = ops.shared_prefix_plan(step["start"], step["lengths"], step["groups"], 8, 2, 64, BF16, DEV)
    q, cache, table, positions = (step[name].to(DEV) for name in ("q", "cache", "table", "positions"))
    run = lambda: ops.attention_shared_prefix(q, cache, table, positions, plan, 8, 2, 64, step["scale"])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        beside = run()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(beside, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        recorded = run()
    for scale in (1.0, 0.5, -1.0):
        q.copy_(step["q"].to(DEV) * scale)
        graph.replay()
        replayed = recorded.clone()
        assert torch.equal(replayed, run())
    

@pytest.mark.parametrize("change", ["heads", "dim", "dtype", "tokens", "table", "sequences", "positions", "scale", "softcap", "sink", "page", "strided"])
def test_refusals(change):
    step = make_step(11, BF16, 8, 2, 64, 16, [(50, 1), (60, 1)], [(0, 2, 40)])
    plan = ops.shared_prefix_plan(step["start"], step["lengths"], step["groups"], 8, 2, 64, BF16, DEV)
    q, cache, table, positions = (step[name].to(DEV) for name in ("q", "cache", "table", "positions"))
    heads, dim, scale, softcap, sink = 8, 64, 0.125, None, None
    if change == "heads":
        heads = 4
    elif change == "dim":
        dim = 32
    elif change == "dtype":
        q = q.float()
    elif change == "tokens":
        q = q[:1].contiguous()
    elif change == "table":
        table = table[:, :2].contiguous()
    elif change == "sequences":
        table = table[:1].contiguous()
    elif change == "positions":
        positions = positions.long()
    elif change == "scale":
        scale = -0.5
    elif change == "softcap":
        softcap = 0.0
    elif change == "sink":
        sink = torch.zeros(4, device=DEV)
    elif change == "page":
        cache = cache[:, :, :, :8 * 64].contiguous()
    elif change == "strided":
        q = torch.cat([q, q], dim=1)[:, :512]
    with pytest.raises(EngineError):
        ops.attention_shared_prefix(q, cache, table, positions, plan, heads, 2, dim, scale, softcap=softcap, sink=sink)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("heads,lengths,prefix", [(4, [49, 81, 50, 17], 48), (40, [49, 81, 50, 17], 47), (64, [65, 97, 66, 1], 64)])
def test_table_entries_of_no_use_are_not_followed(dtype, heads, lengths, prefix):
    """Entries that none of a row's own positions lie on (behind its end, and in the group's other rows the shared blocks) are -1: the
    page before the cache's first, which the buffer around it holds here, with NaN.  Prefixes and ends lie on odd pages of 16 rows, in the middle
    of a block of 32 keys."""
    step = make_step(12, dtype, heads, 2, 64, 16, [(length, 1) for length in lengths], [(0, 3, prefix)])
    want, bound = oracle(step)
    for row, length in enumerate(lengths):
        step["table"][row, (length + 15) // 16:] = -1
        if row in (1, 2):
            step["table"][row, :prefix // 16] = -1
    around = torch.cat([torch.full_like(step["cache"][:1], math.nan), step["cache"]]).to(DEV)
    step["cache"] = around[1:]
    excess = (call(step).double().cpu() - want).abs() - bound
    assert float(excess.max()) <= 0.0


def test_two_calls_at_once():
    """On two streams, each with its own scratch: both have the results that each has alone."""
    steps = [make_step(13 + i, BF16, 32, 4, 64, 16, [(900 + 40 * i + j, 1) for j in range(8)], [(0, 8, 890)]) for i in range(2)]
    on = [{name: step[name].to(DEV) for name in ("q", "cache", "table", "positions")} for step in steps]
    plans = [ops.shared_prefix_plan(step["start"], step["lengths"], step["groups"], 32, 4, 64, BF16, DEV) for step in steps]
    run = lambda i: ops.attention_shared_prefix(on[i]["q"], on[i]["cache"], on[i]["table"], on[i]["positions"], plans[i], 32, 4, 64, 0.125)
    want = [run(0), run(1)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(run(i))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(one, want[i]) for one in got[i])


def test_starts_that_are_not_aligned_are_refused():
    step = make_step(15, BF16, 8, 2, 64, 16, [(50, 1), (60, 1)], [(0, 2, 40)])
    plan = ops.shared_prefix_plan(step["start"], step["lengths"], step["groups"], 8, 2, 64, BF16, DEV)
    q, cache, table, positions = (step[name].to(DEV) for name in ("q", "cache", "table", "positions"))
    shifted = lambda tensor: torch.cat([tensor.flatten()[:1], tensor.flatten()])[1:].view(tensor.shape)
    ops.attention_shared_prefix(q, cache, table, positions, plan, 8, 2, 64, 0.125)
    for first, second in ((shifted(q), cache), (q, shifted(cache))):
        with pytest.raises(EngineError):
            ops.attention_shared_prefix(first, second, table, positions, plan, 8, 2, 64, 0.125)
    for scale, softcap in ((1e-60, None), (math.inf, None), (1.0, 1e-60), (1.0, math.inf), (1e30, 1e-30), (math.nan, None), (1.0, math.nan)):
        with pytest.raises(EngineError):
            ops.attention_shared_prefix(q, cache, table, positions, plan, 8, 2, 64, scale, softcap=softcap)


def test_a_longer_table_of_small_pages_than_a_window_holds():
    """A walk over more than 128 pages, parts that begin on odd pages, and one token alone."""
    check(make_step(16, BF16, 4, 1, 64, 16, [(4500, 1), (4490, 1)], [(0, 2, 4400)]))
    check(make_step(17, BF16, 24, 1, 64, 16, [(4500, 1), (4490, 1)], [(0, 2, 4400)]))
    check(make_step(18, F32, 4, 1, 32, 16, [(4500, 1)], []))


@pytest.mark.parametrize("heads,sequences,groups", [(16, [(300, 1), (310, 1), (290, 1)], [(0, 3, 280)]), (64, [(300, 1), (310, 9), (290, 1)], [(0, 3, 280)])])
def test_pages_past_32_bits(heads, sequences, groups):
    """The step's pages at the end of a cache of more than 2^32 bytes and 2^31 elements: the results of the same pages at its beginning."""
    step = make_step(19, BF16, heads, 8, 64, 32, sequences, groups)
    want = call(step)
    pages, last = step["cache"].shape[0], (1 << 32) // step["cache"][0].numel() + 7
    cache = torch.empty((last + pages, *step["cache"].shape[1:]), dtype=BF16, device=DEV)
    assert cache.numel() > 1 << 32
    cache[last:] = step["cache"].to(DEV)
    step["cache"], step["table"] = cache, step["table"] + last
    assert torch.equal(call(step), want)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 2, 64), (24, 8, 80), (64, 1, 128), (40, 1, 32)])
@pytest.mark.parametrize("softcap", [0.02, 1.0, 50.0, 1000.0, 1030.0, 3e4, 1e6, 1e12, 1e30])
def test_caps_of_any_size(dtype, heads, kv_heads, dim, softcap):
    """A cap far above the scores leaves them as they are: their tangent hyperbolic is then taken of very small numbers."""
    check(make_step(20, dtype, heads, kv_heads, dim, 16, [(150, 1), (170, 3), (133, 1)], [(0, 2, 140)]), softcap)


def test_caps_beyond_what_a_float_tells_apart_are_refused():
    """scale / softcap below the smallest float of 24 bits."""
    step = make_step(21, BF16, 8, 2, 64, 16, [(50, 1), (60, 1)], [(0, 2, 40)])
    plan = ops.shared_prefix_plan(step["start"], step["lengths"], step["groups"], 8, 2, 64, BF16, DEV)
    q, cache, table, positions = (step[name].to(DEV) for name in ("q", "cache", "table", "positions"))
    for scale, softcap in ((1e-3, 2e38), (1e-20, 1e25), (0.125, 1.1e37)):
        with pytest.raises(EngineError):
            ops.attention_shared_prefix(q, cache, table, positions, plan, 8, 2, 64, scale, softcap=softcap)
    ops.attention_shared_prefix(q, cache, table, positions, plan, 8, 2, 64, 0.125, softcap=1e37)
