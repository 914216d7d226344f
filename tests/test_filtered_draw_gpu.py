"""The draw with temperature, top-k, top-p and min-p from given numbers, against its definition in 64 bits (numpy): tokens are
equal, log-probabilities within 2^-24 of their value (the rounding) and 2^-20 (exponentials and differences in 32 bits: 2^-23 each of
what they stand for, a logarithm's error is the relative error of the sum, and a sum of positive terms keeps theirs)."""
import math

import numpy as np
import pytest
import torch

from tlie_amd import ops
from tlie_amd.errors import EngineError

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def oracle(logits, uniform, temperature=None, top_k=None, top_p=None, min_p=None):
    tokens, logprobs = [], []
    for row in range(logits.shape[0]):
        values = logits[row].double().numpy()
        if np.isnan(values).any() or (values == np.inf).any() or (values == -np.inf).all():
            tokens.append(-1), logprobs.append(math.nan)
            continue
        order = np.lexsort((np.arange(values.size), -values))
        with np.errstate(all="ignore"):
            gap = values[order] - values[order[0]]
            t = float(temperature[row]) if temperature is not None else 0.0
            pick = 0
            if t > 0:
                weights = np.where(gap == -np.inf, 0.0, np.exp(np.maximum(gap / t, -800.0)))
                kept = int((weights > 2.0 ** -45).sum())           # (lighter ones are never drawn, as documented)
                if top_k is not None and int(top_k[row]) > 0:
                    kept = min(kept, int(top_k[row]))
                if top_p is not None and float(top_p[row]) < 1.0:
                    sums = np.cumsum(weights[:kept])
                    kept = min(kept, int((sums < float(top_p[row]) * sums[-1]).sum()) + 1)
                if min_p is not None and float(min_p[row]) > 0.0:
                    kept = max(1, int((weights[:kept] >= float(min_p[row])).sum()))
                sums = np.cumsum(weights[:kept])
                u = float(uniform[row])
                pick = min(kept - 1, int((sums <= max(u, 0.0) * sums[-1]).sum())) if u == u else 0
            tokens.append(int(order[pick]))
            logprobs.append(gap[pick] - math.log(np.exp(gap).sum()))
    return np.array(tokens), np.array(logprobs)


def check(logits, uniform, **filters):
    on = lambda value: value.to(DEV) if value is not None else None
    got, logprob = ops.sample_filtered(on(logits), on(uniform), **{name: on(value) for name, value in filters.items()}, logprobs=True)
    want, want_logprob = oracle(logits, uniform, **filters)
    np.testing.assert_array_equal(got.cpu().numpy(), want)
    logprob = logprob.double().cpu().numpy()
    assert (np.isnan(logprob) == np.isnan(want_logprob)).all()
    live = ~np.isnan(want_logprob)
    assert (np.abs(logprob - want_logprob)[live] <= 2.0 ** -24 * np.abs(want_logprob[live]) + 2.0 ** -20).all()
    return got


def rows_of(seed, rows, vocab, spread=2.5):
    gen = torch.Generator().manual_seed(seed)
    logits = spread * torch.randn((rows, vocab), generator=gen)
    logits += (torch.rand((rows, vocab), generator=gen) < 20.0 / vocab) * 8.0 * torch.rand((rows, vocab), generator=gen)
    return logits, torch.rand((rows,), generator=gen), gen


def filters_of(gen, rows):
    choose = lambda values: torch.tensor(values)[torch.randint(0, len(values), (rows,), generator=gen)]
    return dict(temperature=choose([0.0, 0.3, 0.7, 1.0, 1.0, 1.7]), top_k=choose([0, 0, 1, 5, 50, 700, 1 << 30, -1]).int(),
                top_p=choose([1.0, 1.0, 0.99, 0.9, 0.5, 0.01]), min_p=choose([0.0, 0.0, 0.001, 0.05, 0.6]))


@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 2), (40, 5), (64, 255), (64, 1000), (33, 2049), (64, 4097), (200, 8191), (64, 32000), (3, 50261),
                                        (24, 128256), (2, 300001)])
def test_all_filters(rows, vocab):
    logits, uniform, gen = rows_of(vocab, rows, vocab)
    check(logits, uniform, **filters_of(gen, rows))


@pytest.mark.parametrize("name", ["temperature", "top_k", "top_p", "min_p"])
def test_one_filter_at_a_time(name):
    logits, uniform, gen = rows_of(3, 48, 3001)
    filters = filters_of(gen, 48)
    check(logits, uniform, **{"temperature": torch.full((48,), 0.9), name: filters[name]})


def test_without_a_temperature_the_first_maximum():
    logits, uniform, _ = rows_of(4, 9, 700)
    logits[3, 600] = logits[3, 20] = 50.0
    logits[4, 1:4] = 0.0
    logits[4] = -logits[4].abs()
    logits[4, 1], logits[4, 3] = -0.0, 0.0
    got = check(logits, uniform)
    assert got[3] == 20 and got[4] in (1, 2)
    check(logits, uniform, temperature=torch.full((9,), -1.0))


@pytest.mark.parametrize("rounding", ["bfloat16", "halves"])
def test_equal_logits(rounding):
    """Ties go to the lower index, also where top_k and the draw cut through them."""
    logits, uniform, gen = rows_of(5, 64, 9000)
    logits = logits.bfloat16().float() if rounding == "bfloat16" else (logits * 2).round() / 2
    check(logits, uniform, **filters_of(gen, 64))


@pytest.mark.parametrize("vocab", [7, 1000, 20000])
def test_rows_of_one_value(vocab):
    """More tokens of one class than are sorted: the way without a list."""
    logits = torch.zeros(12, vocab)
    logits[4:8, vocab // 2] = -1.0
    uniform = torch.tensor([0.0, 0.25, 0.5, 1 - 2.0 ** -24] * 3)
    k = torch.tensor([0, 3, vocab - 1, 0, 0, 3, vocab - 1, 0, 2500, 2500, 0, 0]).int()
    p = torch.tensor([1.0] * 4 + [0.75] * 4 + [1.0, 0.625, 0.25, 0.4375])
    check(logits, uniform, temperature=torch.ones(12), top_k=k, top_p=p, min_p=torch.tensor([0.0, 0.5] * 6))


@pytest.mark.parametrize("t", [1e-30, 1e-4, 0.05, 5.0, 300.0, 1e20, math.inf])
def test_far_temperatures(t):
    logits, uniform, gen = rows_of(6, 16, 5000)
    filters = filters_of(gen, 16)
    filters["temperature"] = torch.full((16,), t)
    check(logits, uniform, **filters)


def test_numbers_at_the_ends():
    logits, _, _ = rows_of(7, 24, 2500)
    uniform = torch.tensor([0.0, 2.0 ** -24, 0.5, 1 - 2.0 ** -24, 1.0, 1.5, -1.0, math.nan] * 3)
    ones = torch.ones(24)
    check(logits, uniform, temperature=ones, top_p=torch.tensor([1.0, 0.9, 0.0] * 8))
    check(logits, uniform, temperature=ones, top_p=torch.tensor([math.nan, 2.0, -1.0] * 8), min_p=torch.tensor([1.0, 2.0, math.nan, 0.0] * 6))


def test_tokens_that_cannot_be_drawn():
    logits, uniform, gen = rows_of(8, 32, 6000)
    masked = torch.rand((32, 6000), generator=gen) < 0.9
    logits[masked] = -math.inf
    logits[5] = -math.inf
    logits[5, 77] = 3.0
    logits[6] = -math.inf                                           # nothing is left
    logits[7, 9] = math.nan
    logits[8, 9] = math.inf
    logits[9, 10:] = torch.finfo(torch.float32).min
    logits[10] = torch.finfo(torch.float32).min
    logits[10, 5] = torch.finfo(torch.float32).max
    filters = filters_of(gen, 32)
    got = check(logits, uniform, **filters)
    assert got[5] == 77 and got[6] == -1 and got[7] == -1 and got[8] == -1 and got[10] == 5


def test_the_same_row_in_any_batch_and_from_call_to_call():
    logits, uniform, gen = rows_of(9, 300, 7001)
    filters = filters_of(gen, 300)
    got = check(logits, uniform, **filters)
    pick = torch.tensor([7, 299, 0, 31])
    few = ops.sample_filtered(logits[pick].to(DEV), uniform[pick].to(DEV), **{name: value[pick].to(DEV) for name, value in filters.items()})
    assert torch.equal(few.cpu(), got.cpu()[pick])


def test_draws_follow_the_probabilities():
    """A thousand evenly spaced numbers give each token as often as its share says, within one at each end."""
    logits = torch.tensor([0.1, 2.0, -1.0, 1.0, 0.7])
    numbers = (torch.arange(1000) + 0.5) / 1000
    got = ops.sample_filtered(logits.repeat(1000, 1).to(DEV), numbers.to(DEV), torch.ones(1000, device=DEV)).cpu()
    share = torch.softmax(logits.double(), 0)
    for token in range(5):
        assert abs(int((got == token).sum()) - 1000 * float(share[token])) <= 1


def test_outputs_streams_and_replays():
    logits, uniform, gen = rows_of(10, 20, 3000)
    filters = {name: value.to(DEV) for name, value in filters_of(gen, 20).items()}
    logits, uniform = logits.to(DEV), uniform.to(DEV)
    want, want_logprob = ops.sample_filtered(logits, uniform, **filters, logprobs=True)
    out, out_logprob = torch.empty_like(want), torch.empty_like(want_logprob)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.sample_filtered(logits, uniform, **filters, logprobs=True, out=out, out_logprobs=out_logprob)
    torch.cuda.current_stream().wait_stream(side)
    assert got[0] is out and got[1] is out_logprob and torch.equal(out, want) and torch.equal(out_logprob, want_logprob)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        recorded, recorded_logprob = ops.sample_filtered(logits, uniform, **filters, logprobs=True)
    for round in range(3):
        uniform.copy_(torch.rand((20,), generator=gen).to(DEV))
        graph.replay()
        replayed, replayed_logprob = recorded.clone(), recorded_logprob.clone()
        want, want_logprob = ops.sample_filtered(logits, uniform, **filters, logprobs=True)
        assert torch.equal(replayed, want) and torch.equal(replayed_logprob, want_logprob)


def test_refusals_and_no_rows():
    logits, uniform = torch.zeros(4, 10, device=DEV), torch.zeros(4, device=DEV)
    assert ops.sample_filtered(logits[:0], uniform[:0]).shape == (0,)
    bad = [dict(logits=logits.bfloat16()), dict(logits=logits[0]), dict(logits=logits[:, :0]), dict(logits=torch.zeros(10, 4, device=DEV).t()), dict(uniform=None),
           dict(uniform=uniform.double()), dict(uniform=uniform[:3]), dict(uniform=uniform.cpu()), dict(top_k=torch.zeros(4, device=DEV)),
           dict(top_p=torch.zeros(5, device=DEV)), dict(min_p=torch.zeros(4, 1, device=DEV)), dict(temperature=torch.ones(4, dtype=torch.float64, device=DEV)),
           dict(out=torch.zeros(4, device=DEV)), dict(out_logprobs=uniform)]
    for change in bad:
        with pytest.raises(EngineError):
            ops.sample_filtered(**{"logits": logits, "uniform": uniform, **change})


@pytest.mark.parametrize("rows,vocab", [(2, 60000), (20, 3000)])
def test_two_calls_at_once_and_replays_beside_eager_calls(rows, vocab):
    """Both forms (a row in parts, a row by one workgroup) on two streams, and in a recording with eager calls between its replays."""
    logits, uniform, gen = rows_of(11, rows, vocab)
    filters = {name: value.to(DEV) for name, value in filters_of(gen, rows).items()}
    logits, uniform = logits.to(DEV), uniform.to(DEV)
    inputs = [(logits, uniform), (logits.flip(0).contiguous(), uniform.flip(0).contiguous())]
    run = lambda i: ops.sample_filtered(*inputs[i], **filters, logprobs=True)
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
        for tokens, logprobs in got[i]:
            assert torch.equal(tokens, want[i][0]) and torch.equal(logprobs, want[i][1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        recorded = run(0)
    for _ in range(4):
        uniform.copy_(torch.rand((rows,), generator=gen).to(DEV))
        graph.replay()
        replayed = [value.clone() for value in recorded]
        run(1)
        eager = run(0)
        assert torch.equal(replayed[0], eager[0]) and torch.equal(replayed[1], eager[1])


def test_rows_that_start_anywhere():
    """Rows of a vocabulary that is no multiple of four, in a tensor that itself starts past such a place."""
    for offset in (1, 2, 3):
        logits, uniform, gen = rows_of(12 + offset, 5, 30001)
        filters = {name: value.to(DEV) for name, value in filters_of(gen, 5).items()}
        shifted = torch.cat([torch.full((offset,), math.inf), logits.flatten(), torch.full((3,), math.inf)]).to(DEV)[offset:offset + logits.numel()].view(logits.shape)
        want = ops.sample_filtered(logits.to(DEV), uniform.to(DEV), **filters, logprobs=True)
        got = ops.sample_filtered(shifted, uniform.to(DEV), **filters, logprobs=True)
        assert torch.equal(got[0], want[0])
        check(logits, uniform, **{name: value.cpu() for name, value in filters.items()})


def test_more_logits_than_32_bits_count():
    """Rows past the 2^31st element (8.6 GB): the last rows draw what they draw alone."""
    rows, vocab = 65535, 32800
    logits = torch.zeros((rows, vocab), device=DEV)
    few, uniform, gen = rows_of(16, 8, vocab)
    filters = {name: value.to(DEV) for name, value in filters_of(gen, 8).items()}
    logits[-8:] = few.to(DEV)
    numbers = torch.zeros(rows, device=DEV)
    numbers[-8:] = uniform.to(DEV)
    spread = {"temperature": torch.zeros(rows, device=DEV), "top_k": torch.zeros(rows, dtype=torch.int32, device=DEV),
              "top_p": torch.ones(rows, device=DEV), "min_p": torch.zeros(rows, device=DEV)}
    for name, value in spread.items():
        value[-8:] = filters[name]
    got = ops.sample_filtered(logits, numbers, **spread)
    assert torch.equal(got[-8:], ops.sample_filtered(few.to(DEV), uniform.to(DEV), **filters))
    assert not got[:-8].any()


@pytest.mark.parametrize("rows,vocab", [(3, 1001), (3, 1002), (2, 60001), (2, 60003)])
def test_the_first_of_equal_maxima_wherever_they_stand(rows, vocab):
    """The largest logit at two places, one of them in the last, cut group of four tokens, the other at every place of the first
    groups; also with rows that start past a multiple of 16 bytes (every row but the first of an odd vocabulary)."""
    places = list(range(12)) + [511 * 4, 512 * 4, vocab // 2, vocab - 2]
    for place in places:
        if place >= vocab - 1:
            continue
        logits = torch.zeros((rows, vocab))
        logits[:, place], logits[:, vocab - 1] = 3.0, 3.0
        zero = torch.zeros(rows, device=DEV)
        got = ops.sample_filtered(logits.to(DEV), zero)
        assert got.tolist() == [place] * rows, place
        got = ops.sample_filtered(logits.to(DEV), zero, torch.full((rows,), 0.1, device=DEV), top_k=torch.ones(rows, dtype=torch.int32, device=DEV))
        assert got.tolist() == [place] * rows, place


def test_the_largest_vocabulary():
    """Tokens at both ends of 2^24 - 1, with weights of 2^-38 of the largest at the least."""
    vocab = ops.DRAW_MAX_VOCAB
    logits = torch.full((3, vocab), -60.0)
    logits[:, 5], logits[:, vocab - 1], logits[:, vocab // 2] = 2.0, 1.0, 0.0
    logits[2, vocab - 2] = 3.0
    uniform = torch.tensor([0.1, 0.7, 0.99])
    check(logits, uniform, temperature=torch.ones(3), top_k=torch.tensor([0, 2, 3], dtype=torch.int32), min_p=torch.full((3,), 0.01))
    with pytest.raises(EngineError):
        ops.sample_filtered(torch.zeros((1, vocab + 1), device=DEV), torch.zeros(1, device=DEV))


@pytest.mark.parametrize("rows,vocab", [(1, 20000), (1, 28000), (3, 20480), (35, 24576)])
def test_odd_numbers_of_rows_times_parts(rows, vocab):
    assert rows * ops.draw_parts(rows, vocab) % 2 == 1
    logits, uniform, gen = rows_of(vocab + rows, rows, vocab)
    check(logits, uniform, **filters_of(gen, rows))
    check(logits, uniform, temperature=torch.full((rows,), 0.8), top_p=torch.full((rows,), 0.9))


@pytest.mark.parametrize("rows,vocab", [(6, 3000), (2, 60000), (6, 20000)])
def test_min_p_above_one_keeps_the_first_token_alone(rows, vocab):
    """No weight reaches more than the largest's, so of several largest the first is kept; at 1 they all are.  Also where more tokens
    are equal than are sorted."""
    logits, _, gen = rows_of(vocab, rows, vocab)
    logits[:, [40, 700, vocab - 1]] = 30.0
    logits[1] = 2.0
    ones = torch.ones(rows)
    for min_p in (1.0, 1.0 + 2.0 ** -23, 1.5, 1e30, math.inf):
        for u in (0.0, 0.4, 0.99):
            got = check(logits, u * ones, temperature=0.8 * ones, min_p=min_p * ones)
            assert min_p == 1.0 or got.tolist() == [40, 0] + [40] * (rows - 2)


@pytest.mark.parametrize("rows,vocab", [(7, 1001), (7, 4098), (2, 60003)])
def test_rows_that_have_to_be_finite(rows, vocab):
    """With finite=True one logit of -inf, at any place of the row, gives -1; the other rows draw what they draw without."""
    logits, uniform, _ = rows_of(vocab, rows, vocab)
    on = lambda value: value.to(DEV)
    draw = lambda values, **named: ops.sample_filtered(on(values), on(uniform), torch.ones(rows, device=DEV), torch.full((rows,), 9, dtype=torch.int32, device=DEV),
                                                       logprobs=True, **named)
    want, want_logprobs = draw(logits)
    got, logprobs = draw(logits, finite=True)
    assert torch.equal(got, want) and torch.equal(logprobs, want_logprobs)
    for place in (0, 1, 2, 3, 4, 500, vocab // 2, vocab - 4, vocab - 3, vocab - 2, vocab - 1):
        masked = logits.clone()
        masked[1, place] = -math.inf
        assert draw(masked)[0][1] >= 0
        got, logprobs = draw(masked, finite=True)
        assert got[1] == -1 and math.isnan(logprobs[1]), place
        assert torch.equal(got[[0] + list(range(2, rows))], want[[0] + list(range(2, rows))])


@pytest.mark.parametrize("gap", [4.0, 8.3, 9.7, 11.9, 13.7])
@pytest.mark.parametrize("rows,vocab", [(3, 200003), (40, 33000)])
def test_log_probabilities_of_mass_far_below_the_maximum(rows, vocab, gap):
    """One high logit, and most of the weight (or as much as the vocabulary holds) at a gap below it.  A term of the sum is off by (2 + 1.2 gap)
    2^-23 of it (the difference's and the product's roundings 2^-24 of the gap each, log2(e)'s own 2^-26; an exponential and a sum of four 2^-23
    each), the sum by the mean of these by weight; the logarithm's error is the sum's relative one, and the result is rounded to 2^-24 of it."""
    gen = torch.Generator().manual_seed(vocab)
    logits = 3.0 - gap + 0.3 * torch.randn((rows, vocab), generator=gen).clamp(-3, 3)
    logits[:, 17] = 3.0 + torch.rand((rows,), generator=gen)
    uniform, temperature = torch.rand((rows,), generator=gen), torch.where(torch.arange(rows) % 3 == 0, 0.0, 1.0)
    tokens, logprobs = ops.sample_filtered(logits.to(DEV), uniform.to(DEV), temperature.to(DEV), logprobs=True)
    wide = logits.double()
    below = wide.max(dim=1, keepdim=True).values - wide
    weights = torch.exp(-below)
    mean = (weights * below).sum(dim=1) / weights.sum(dim=1)
    want = torch.log_softmax(wide, dim=1).gather(1, tokens.cpu().long().unsqueeze(1)).squeeze(1)
    bound = (2.0 + 1.2 * mean) * 2.0 ** -23 + 2.0 ** -24 * want.abs()
    assert float(((logprobs.double().cpu() - want).abs() - bound).max()) <= 0.0


@pytest.mark.parametrize("t", [1e-3, 1.0, 1e10, 1e18, 1e20, 1e37, math.inf])
@pytest.mark.parametrize("rows,vocab", [(9, 900), (9, 4000), (2, 60000)])
def test_min_p_of_one_at_any_temperature(rows, vocab, t):
    """Kept is what weighs as much as the largest in 64 bits: equal logits, and at a temperature beyond 10^17 times the logits all of them."""
    logits, _, gen = rows_of(vocab + 5, rows, vocab)
    logits[:, [3, 600]] = 25.0
    ones = torch.ones(rows)
    for u in (0.0, 0.3, 0.77, 0.999):
        check(logits, u * ones, temperature=t * ones, min_p=ones)
        check(logits, u * ones, temperature=t * ones, min_p=ones, top_p=0.7 * ones, top_k=torch.full((rows,), 300).int())
        check(logits, u * ones, temperature=t * ones, min_p=(1 - 2.0 ** -24) * ones)


@pytest.mark.parametrize("t", [1.0, 1e18, 1e24, math.inf])
def test_min_p_above_one_at_any_temperature(t):
    logits, uniform, _ = rows_of(77, 24, 3000)
    got = check(logits, uniform, temperature=torch.full((24,), t), min_p=torch.full((24,), 1.5))
    assert torch.equal(got.cpu().long(), logits.argmax(dim=1))


@pytest.mark.parametrize("t", [2.0 ** 42, 2.0 ** 46, 2.0 ** 50, 2.0 ** 54])
@pytest.mark.parametrize("rows,vocab", [(9, 700), (9, 3000), (2, 60000)])
def test_min_p_of_one_where_some_weights_are_the_largests_in_64_bits(rows, vocab, t):
    """Gaps of x T 2^-54: exp(-x 2^-54) = 1 - x 2^-54 (the square is below 2^-100) lies x / 2 of a step of 2^-53 below 1, and is 1 when rounded for
    x < 1 and less for x > 1.  So what is kept, with equal weights, is known without an exponential (numpy's gives less than 1 from
    x = 0.9 on), and the token is the first of which more than u of them stand no later."""
    gen = torch.Generator().manual_seed(vocab)
    steps = torch.randint(1, 40, (rows, vocab), generator=gen).double() + 0.25
    steps[:, 11] = 0.0
    fewer = steps * 0.3
    fewer[:, 12] = 1.2
    for x, k in ((steps, 0), (steps, 5), (fewer, 0), (fewer, 17)):
        logits = (-x * (t * 2.0 ** -54)).float()                  # (x of few bits, or rounded to 2^-24 of it: none near 1 but 0.975 and 1.275)
        order = np.lexsort((np.broadcast_to(np.arange(vocab), (rows, vocab)), -logits.numpy()), axis=1)
        for u in (0.0, 0.3, 0.77, 0.999):
            number = float(np.float32(u))
            want = []
            for row in range(rows):
                kept = int((x[row] < 1.0).sum())
                kept = min(kept, k) if k else kept
                want.append(order[row, min(kept - 1, int(number * kept))])
            ones = torch.ones(rows, device=DEV)
            got = ops.sample_filtered(logits.to(DEV), number * ones, t * ones, min_p=ones,
                                      top_k=torch.full((rows,), k, dtype=torch.int32, device=DEV))
            np.testing.assert_array_equal(got.cpu().numpy(), np.array(want))
