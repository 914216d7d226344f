"""The work list of attention over shared prefixes: every (token, head, key) in exactly one item, every part written once; and
what the plan refuses."""
import random

import numpy as np
import pytest
import torch

from tlie_amd import ops
from tlie_amd.errors import EngineError


def drawn_step(rng):
    """Cumulative token counts, lengths, groups and every sequence's prefix."""
    sequences = rng.randint(0, 12)
    counts = [rng.choice([0, 1, 1, 1, rng.randint(1, 40)]) for _ in range(sequences)]
    groups, prefix, at = [], [0] * sequences, 0
    while at < sequences:
        count = rng.randint(1, 4)
        if rng.random() < 0.6 and at + count <= sequences:
            groups.append((at, count, rng.choice([0, 1, 16, 100, 1000, 5000])))
            prefix[at:at + count] = [groups[-1][2]] * count
            at += count
        else:
            at += 1
    lengths = [prefix[s] + counts[s] + rng.choice([0, 1, 50, 1000]) if counts[s] else rng.randint(0, 100) for s in range(sequences)]
    rng.shuffle(groups)
    return np.concatenate([[0], np.cumsum(counts)]).astype(np.int64), np.array(lengths, dtype=np.int64), groups, prefix


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads,kv_heads,dim", [(32, 4, 64), (32, 8, 128), (8, 8, 256), (40, 1, 64), (12, 4, 48)])
def test_every_key_of_every_column_is_in_one_item(heads, kv_heads, dim, dtype):
    rng, group = random.Random(heads), heads // kv_heads
    for _ in range(40):
        start, lengths, groups, prefix = drawn_step(rng)
        items, part_first = ops.shared_prefix_items(start, lengths, groups, heads, kv_heads, dim, dtype)
        covered, written = {}, set()
        for sequence, tok0, tokens, col0, low, high, own, part in items.tolist():
            assert low < high
            for column in range(col0, min(col0 + ops.prefix_tile_columns(tokens * group - col0, dim, dtype), tokens * group)):
                token, head = tok0 + column // group, column % group
                seq = int(np.searchsorted(start, token, side="right") - 1)
                position = lengths[seq] - start[seq + 1] + token
                assert (seq == sequence and low >= prefix[seq]) if own else high <= prefix[seq]
                end = min(high, position + 1) if own else high
                if part < part_first[token + 1] - part_first[token]:
                    assert (part_first[token] + part, head) not in written
                    written.add((part_first[token] + part, head))
                    covered.setdefault((token, head), []).append((low, max(low, end)))
                else:
                    assert end <= low                          # nothing the token sees
        for token in range(int(start[-1])):
            seq = int(np.searchsorted(start, token, side="right") - 1)
            for head in range(group):
                end = 0
                for low, high in sorted(covered[token, head]):
                    assert low == end or high == low
                    end = max(end, high)
                assert end == lengths[seq] - start[seq + 1] + token + 1
                assert all((part, head) in written for part in range(part_first[token], part_first[token + 1]))


@pytest.mark.parametrize("start,lengths,groups,heads", [
    ([0, 1], [1, 1], [], 8),                       # lengths of another count
    ([1, 2], [4], [], 8),                          # not from 0
    ([0, 2, 1], [4, 4], [], 8),                    # counting down
    ([0, 3], [2], [], 8),                          # shorter than what it brings
    ([0, 1, 2], [9, 9], [(0, 2, 9)], 8),           # a token inside its prefix
    ([0, 1, 2], [9, 9], [(0, 2, 4), (1, 1, 4)], 8),     # a sequence in two groups
    ([0, 1, 2], [9, 9], [(1, 2, 4)], 8),           # a group past the step
    ([0, 1, 2], [9, 9], [(0, 0, 4)], 8),           # a group of none
    ([0, 1, 2], [9, 9], [(0, 2, -1)], 8),          # a negative prefix
    ([0, 1, 2], [9, 9], [], 9),                    # heads that do not share kv heads evenly
    ([0, 1], [(1 << 30) + 1], [], 8),              # positions whose blocks a kernel cannot count in 32 bits
])
def test_plans_that_are_refused(start, lengths, groups, heads):
    with pytest.raises(EngineError):
        ops.shared_prefix_plan(start, lengths, groups, heads, 4, 64, torch.bfloat16, "cpu")


def test_a_prefix_is_read_through_a_sequence_that_holds_it():
    items, part_first = ops.shared_prefix_items([0, 0, 1, 2], [3, 9, 12], [(0, 3, 4)], 8, 4, 64, torch.bfloat16)
    assert items[items[:, 6] == 0][:, 0].tolist() == [1] and part_first.tolist() == [0, 2, 4]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads,kv_heads,dim", [(32, 4, 64), (32, 8, 128), (8, 8, 256), (40, 1, 64), (150, 1, 128), (12, 4, 48)])
def test_a_recorded_plan_holds_any_step_of_single_tokens(heads, kv_heads, dim, dtype):
    """Cut into one part each, which is what it comes down to when more do not fit."""
    rng = random.Random(dim)
    for tokens in (1, 2, 3, 8, 16, 33, 64, 256):
        items_held, parts_held = ops.RecordedPrefixPlan.room(tokens, heads, kv_heads, dim, dtype)
        for largest in (2, 3, tokens):
            groups, at, lengths = [], 0, []
            while at < tokens:
                count = min(tokens - at, rng.randint(2, max(2, largest)))
                prefix = rng.choice([1, 100, 20000])
                groups.append((at, count, prefix))
                lengths += [prefix + rng.choice([1, 700, 9000]) for _ in range(count)]
                at += count
            items, part_first = ops.shared_prefix_items(range(tokens + 1), lengths, groups, heads, kv_heads, dim, dtype, 256, 1)
            assert items.shape[0] <= items_held and part_first[-1] <= parts_held


def test_other_types_are_refused():
    with pytest.raises(EngineError):
        ops.shared_prefix_plan([0, 1], [4], [], 8, 4, 64, torch.float16, "cpu")


def test_arguments_on_the_host_are_refused():
    logits, number = torch.zeros(2, 8), torch.zeros(2)
    with pytest.raises(EngineError):
        ops.sample_filtered(logits, number)
    plan = ops.SharedPrefixPlan(torch.zeros(1, 8, dtype=torch.int32), torch.zeros(2, dtype=torch.int32), 1, 1, 1, 1, (2, 1, 16, torch.float32))
    with pytest.raises(EngineError):
        ops.attention_shared_prefix(torch.zeros(1, 32), torch.zeros(1, 2, 1, 256), torch.zeros(1, 1, dtype=torch.int32),
                                    torch.zeros(1, dtype=torch.int32), plan, 2, 1, 16, 1.0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads,kv_heads,dim", [(32, 4, 64), (4, 2, 16), (40, 1, 64), (12, 4, 48)])
def test_the_items_of_short_steps_cover_every_column_once(heads, kv_heads, dim, dtype):
    rng, group, short = random.Random(dim), heads // kv_heads, 0
    for _ in range(60):
        start, lengths, groups, prefix = drawn_step(rng)
        items = ops.direct_prefix_items(start, lengths, groups, heads, kv_heads, dim, dtype, 256)
        if items is None:
            continue
        short += 1
        assert items.shape[0] * kv_heads <= 256
        seen = set()
        for sequence, tok0, tokens, col0, shared, end, own, reader in items.tolist():
            assert own == 1 and tok0 == start[sequence] and tokens == start[sequence + 1] - start[sequence] and shared == prefix[sequence]
            assert lengths[reader] >= shared and (reader == sequence or any(a <= reader <= sequence < a + b for a, b, _ in groups))
            for column in range(col0, min(col0 + 16, tokens * group)):
                seen.add((sequence, column))
                assert end > lengths[sequence] - tokens + column // group        # the token's own key is among them
        assert len(seen) == int(start[-1]) * group
    assert short > 0


def test_long_steps_and_wide_heads_are_cut():
    plan = lambda length, dim, dtype=torch.bfloat16, count=4: ops.direct_prefix_items(range(count + 1), [length] * count, [(0, count, length - 1)], 32, 4, dim, dtype, 256)
    assert plan(700, 64) is not None and plan(1000, 64) is None
    assert plan(300, 64, torch.float32) is not None and plan(700, 64, torch.float32) is None
    assert plan(100, 128) is None and plan(100, 64, count=65) is None


@pytest.mark.parametrize("start,lengths,fits", [
    ([0, 1, 2], [64, 64], True), ([0, 1, 2, 3, 4], [10, 20, 64, 3], True),
    ([0, 1, 2], [64, 65], False),                     # longer than the tables that the plan goes with
    ([0, 1, 1], [3, 1000], False),                    # the same, of a sequence that brings nothing
    ([0, 1, 1, 1, 1, 2], [9, 9, 9, 9, 9], False),     # more sequences than such tables have rows
    ([0, 1, 2, 3, 4, 5], [9] * 5, False),             # more tokens
])
def test_steps_beyond_a_recorded_plan_are_refused(start, lengths, fits):
    """A recorded step's block table is checked against what its plan may hold, once; so `fill` keeps every step within that."""
    plan = ops.RecordedPrefixPlan(4, 64, 8, 4, 64, torch.bfloat16, "cpu")
    if fits:
        plan.fill(start, lengths, [])
        items, _ = ops.shared_prefix_items(start, lengths, [], 8, 4, 64, torch.bfloat16)
        assert plan.plan.items[:len(items)].tolist() == items.tolist() and not plan.plan.items[len(items):].any()
    else:
        before = plan.plan.items.clone()
        with pytest.raises(EngineError):
            plan.fill(start, lengths, [])
        assert torch.equal(plan.plan.items, before)


def test_a_recorded_plans_buffer_is_written_behind_its_last_transfer():
    """`fill` again, with no step in between: the host's buffer is still being read until the event behind its transfer has been reached."""
    log = []

    class Event:
        def synchronize(self):
            log.append(("wait", plan._host.clone()))

        def record(self):
            log.append(("record", plan._host.clone()))
    plan = ops.RecordedPrefixPlan(4, 64, 8, 4, 64, torch.bfloat16, "cpu")
    plan._sent = Event()
    plan.fill([0, 1, 2], [40, 41], [(0, 2, 39)])
    plan.fill([0, 1], [17], [])
    assert [name for name, _ in log] == ["wait", "record", "wait", "record"]
    assert torch.equal(log[1][1], log[2][1]) and not torch.equal(log[2][1], log[3][1])


@pytest.mark.parametrize("start,lengths", [([0, 1 << 40], [1 << 40]), ([0, 1 << 62], [1 << 62]), ([0, 1 << 26], [1 << 27])])
def test_more_tokens_than_a_launch_takes_are_refused_and_not_allocated(start, lengths):
    with pytest.raises(EngineError):
        ops.shared_prefix_plan(start, lengths, [], 8, 4, 64, torch.bfloat16, "cpu")


def recorded(tokens, start, lengths, groups, sizes):
    plan = ops.RecordedPrefixPlan(tokens, 1 << max(int(length) for length in lengths).bit_length(), *sizes, "cpu")
    plan.fill(start, lengths, groups)
    return plan.plan


@pytest.mark.parametrize("heads,kv_heads,count,prefix", [(32, 8, 24, 30000), (32, 8, 32, 20000), (32, 8, 32, 30000), (32, 8, 64, 20000), (32, 8, 64, 30000),
                                                         (8, 1, 32, 12000), (32, 4, 64, 30000), (32, 32, 16, 30000)])
def test_recorded_steps_are_cut_as_others_are(heads, kv_heads, count, prefix):
    lengths = [prefix + 1 + 37 * i % 300 for i in range(count)]
    start, sizes = range(count + 1), (heads, kv_heads, 128, torch.bfloat16)
    items, part_first = ops.shared_prefix_items(start, lengths, [(0, count, prefix)], *sizes)
    plan = recorded(1 << (count - 1).bit_length(), start, lengths, [(0, count, prefix)], sizes)
    assert plan.items[:len(items)].tolist() == items.tolist() and not plan.items[len(items):].any()
    assert plan.part_first[:count + 1].tolist() == part_first.tolist()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads,kv_heads,dim", [(32, 4, 64), (32, 8, 128), (8, 8, 256), (40, 1, 64), (150, 1, 128), (12, 4, 48), (8, 1, 128), (32, 32, 128)])
def test_recorded_steps_of_any_groups_are_cut_as_others_are(heads, kv_heads, dim, dtype):
    """Groups of two sequences or more, others beside them, prefixes and own keys of any length."""
    rng = random.Random(heads + dim)
    for tokens in (1, 2, 4, 8, 16, 32, 64, 128, 256):
        for _ in range(4):
            count, groups, lengths = rng.randint(tokens // 2 + 1, tokens), [], []
            while len(lengths) < count:
                members = min(count - len(lengths), rng.choice([1, 2, 3, 8, count]))
                prefix = int(2 ** rng.uniform(4, 15)) if members > 1 else 0
                if members > 1:
                    groups.append((len(lengths), members, prefix))
                lengths += [prefix + int(2 ** rng.uniform(0, rng.choice([4, 9, 13]))) for _ in range(members)]
            items, part_first = ops.shared_prefix_items(range(count + 1), lengths, groups, heads, kv_heads, dim, dtype)
            plan = recorded(tokens, range(count + 1), lengths, groups, (heads, kv_heads, dim, dtype))
            assert plan.items[:len(items)].tolist() == items.tolist() and not plan.items[len(items):].any()
            assert plan.part_first[:count + 1].tolist() == part_first.tolist() and plan.parts >= part_first[-1]


def test_a_recorded_plan_that_is_short_is_cut_as_finely_as_it_holds(monkeypatch):
    """Not by halves: 33 parts of a prefix for room of 33 a token and one of its own each."""
    count, prefix, sizes = 32, 30000, (32, 8, 128, torch.bfloat16)
    lengths = [prefix + 1 + i for i in range(count)]
    monkeypatch.setattr(ops.RecordedPrefixPlan, "room", staticmethod(lambda *sizes: (300, 34 * count)))
    plan = recorded(count, range(count + 1), lengths, [(0, count, prefix)], sizes)
    best = max(most for most in range(1, 65) if ops.shared_prefix_items(range(count + 1), lengths, [(0, count, prefix)], *sizes, 256, most)[1][-1] <= 34 * count)
    items, part_first = ops.shared_prefix_items(range(count + 1), lengths, [(0, count, prefix)], *sizes, 256, best)
    assert 24 < best < 64 and plan.items[:len(items)].tolist() == items.tolist() and plan.part_first[:count + 1].tolist() == part_first.tolist()
    monkeypatch.setattr(ops.RecordedPrefixPlan, "room", staticmethod(lambda *sizes: (300, count)))
    with pytest.raises(EngineError):
        recorded(count, range(count + 1), lengths, [(0, count, prefix)], sizes)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads,kv_heads,dim", [(32, 4, 64), (32, 8, 128), (8, 8, 256), (40, 1, 64), (12, 4, 48), (24, 8, 80), (64, 8, 64)])
def test_recorded_steps_of_portions_are_cut_as_others_are(heads, kv_heads, dim, dtype):
    """Families that decode, or bring portions, beside others' portions; sequences beyond the step's bring nothing."""
    rng = random.Random(heads + dim)
    for tokens in (16, 64, 256, 512):
        for sequences in (8, min(64, tokens)):
            for _ in range(4):
                left, counts, lengths, groups = tokens, [], [], []
                while left > 0 and len(counts) < sequences:
                    members = min(sequences - len(counts), rng.choice([1, 2, 5, sequences]), left)
                    prefix = int(2 ** rng.uniform(4, 15)) if members > 1 else 0
                    if members > 1:
                        groups.append((len(counts), members, prefix))
                    for _ in range(members):
                        counts.append(1 if rng.random() < 0.6 else rng.randint(1, max(1, left // 2)))
                        counts[-1] = min(counts[-1], left)
                        left -= counts[-1]
                        lengths.append(prefix + counts[-1] + int(2 ** rng.uniform(0, rng.choice([4, 9, 13]))))
                start = np.concatenate([[0], np.cumsum(counts)])
                items, part_first = ops.shared_prefix_items(start, lengths, groups, heads, kv_heads, dim, dtype)
                padded = np.concatenate([start, np.full(sequences - len(counts), start[-1])]), lengths + [1] * (sequences - len(counts))
                plan = ops.RecordedPrefixPlan(tokens, 1 << max(lengths).bit_length(), heads, kv_heads, dim, dtype, "cpu", sequences)
                plan.fill(*padded, groups)
                plan = plan.plan
                assert plan.sequences == sequences and plan.items[:len(items)].tolist() == items.tolist() and not plan.items[len(items):].any()
                assert plan.part_first[:start[-1] + 1].tolist() == part_first.tolist() and (plan.part_first[start[-1]:] == part_first[-1]).all()
                assert plan.parts >= part_first[-1]


@pytest.mark.parametrize("heads,groups,count,prefix,portion,dtype,pays", [
    ((4, 64), 1, 64, 500, 0, torch.bfloat16, False), ((4, 64), 1, 64, 1000, 0, torch.bfloat16, True), ((4, 64), 8, 8, 1000, 0, torch.bfloat16, True),
    ((4, 64), 8, 8, 500, 0, torch.bfloat16, False), ((4, 64), 1, 32, 2000, 0, torch.bfloat16, True), ((4, 64), 1, 8, 2000, 0, torch.bfloat16, False),
    ((8, 128), 1, 64, 250, 0, torch.bfloat16, False), ((8, 128), 1, 64, 500, 0, torch.bfloat16, True), ((8, 128), 16, 4, 250, 0, torch.bfloat16, False),
    ((8, 128), 1, 16, 500, 0, torch.bfloat16, True), ((8, 128), 1, 8, 1000, 0, torch.bfloat16, True), ((8, 128), 1, 2, 8000, 0, torch.bfloat16, True),
    ((32, 64), 1, 64, 250, 0, torch.bfloat16, False), ((8, 80), 1, 64, 500, 0, torch.bfloat16, False), ((8, 80), 1, 64, 1000, 0, torch.bfloat16, True),
    ((8, 64), 1, 64, 250, 0, torch.float32, True), ((8, 64), 1, 64, 500, 0, torch.float32, True), ((8, 128), 1, 64, 250, 0, torch.float32, True),
    ((4, 64), 1, 4, 300, 0, torch.float32, False),
    ((4, 64), 1, 32, 2000, 2000, torch.bfloat16, False), ((4, 64), 1, 64, 2000, 636, torch.bfloat16, True), ((4, 64), 1, 32, 2000, 1000, torch.bfloat16, False),
    ((4, 64), 1, 16, 6000, 2000, torch.bfloat16, True), ((8, 128), 1, 32, 2000, 2000, torch.bfloat16, True), ((8, 128), 1, 32, 1500, 2000, torch.bfloat16, False),
    ((4, 64), 1, 64, 400, 256, torch.bfloat16, True), ((4, 64), 1, 32, 2000, 2000, torch.float32, True)])
def test_steps_take_the_faster_attention(heads, groups, count, prefix, portion, dtype, pays):
    """Measured on both sides of each line, families that decode, alone or beside another prompt's portion."""
    of = [(group * count, count, prefix) for group in range(groups)]
    assert ops.shared_prefix_pays(of, *heads, dtype, groups * count + portion if portion else 0) is pays


def test_many_short_groups_count_as_their_sum():
    groups = [(4 * i, 4, 1200) for i in range(8)]
    assert ops.shared_prefix_pays(groups, 8, 128) and not ops.shared_prefix_pays(groups[:1], 8, 128)
