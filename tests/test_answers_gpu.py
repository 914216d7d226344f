"""Several answers to a prompt through the engine: forked requests, recorded and unrecorded steps that read a shared prefix once,
draws with top_k and min_p, log-probabilities, the command line."""
import json
import math

import pytest
import torch

from gpu_helpers import CONFIG_A, CONFIG_B, CUT_TOLERANCE, make_model, random_tokens
from tlie_amd import Engine, StepEntry, ops
from tlie_amd.engine.scheduler import SamplingParams

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
# one layer whose caches are wide enough that reading a prefix of some hundred positions once pays by itself
CONFIG_WIDE = dict(CONFIG_A, hidden_size=128, intermediate_size=128, num_hidden_layers=1, num_attention_heads=16, num_key_value_heads=8, head_dim=128,
                   max_position_embeddings=1024)


@pytest.fixture
def always_shared(monkeypatch):
    monkeypatch.setattr("tlie_amd.engine.step.ops_shared_prefix_pays", lambda *sizes: True)


@pytest.fixture
def counted(monkeypatch):
    calls = []
    real = ops.attention_shared_prefix

    def call(*args, **named):
        calls.append(args[0].shape[0])
        return real(*args, **named)
    monkeypatch.setattr(ops, "attention_shared_prefix", call)
    return calls


@pytest.mark.parametrize("config", [CONFIG_A, CONFIG_B])
def test_answers_are_those_of_separate_requests(tmp_path, config, always_shared, counted):
    folder = make_model(tmp_path / "m", config, 5, "float32")
    prompts = [random_tokens(1, 70, 256), random_tokens(2, 41, 256), random_tokens(3, 5, 256)]
    options = dict(max_tokens=12, temperature=0.9, top_p=0.95, seed=11)
    engine = Engine(folder, dtype="float32", max_tokens=2048, max_requests=16)
    got = engine.generate(prompts, answers=4, **options)
    assert counted and engine.cache.free_pages() == [engine.cache.num_pages]
    engine.cache.check()
    plain = Engine(folder, dtype="float32", max_tokens=2048, max_requests=16)
    counted.clear()
    want = plain.generate([prompt for prompt in prompts for _ in range(4)], **options)
    assert not counted
    assert got == [want[0:4], want[4:8], want[8:12]]
    # and again, by the recordings that are there now
    assert engine.generate(prompts, answers=4, **options) == got


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_a_step_over_a_shared_prefix(tmp_path, dtype, always_shared, counted):
    """Logits of forked requests against those of requests that computed the prompt themselves; recorded, launched one by one on
    the recording's arrays, and unrecorded."""
    folder = make_model(tmp_path / "m", CONFIG_B, 6, dtype)
    prompt = random_tokens(4, 90, 512)
    outputs = {}
    for name, options in (("recorded", {}), ("laid out", dict(capture_graphs=False)), ("plain", dict(use_graphs=False)), ("apart", {})):
        engine = Engine(folder, dtype=dtype, max_tokens=2048, max_requests=8, **options)
        engine.admit("a")
        engine.step([StepEntry("a", prompt[:-1], [])])
        for request in "bcd":
            if name == "apart":
                engine.admit(request)
                engine.step([StepEntry(request, prompt[:-1], [])])
            else:
                engine.cache.fork("a", request, len(prompt) - 1)
        counted.clear()
        logits = []
        for turn in range(4):                            # (a recording is made by the first, replayed by the others)
            tokens = [prompt[-1]] * 4 if turn == 0 else [7 * turn, 7 * turn + 1, 3, 200 + turn]
            logits.append(engine.step([StepEntry(request, [token], [0]) for request, token in zip("abcd", tokens)]))
        assert bool(counted) == (name != "apart")
        outputs[name] = torch.stack(logits).double().cpu()
    assert torch.equal(outputs["recorded"], outputs["laid out"])
    scale = outputs["apart"].abs().amax(dim=-1, keepdim=True)
    tolerance = 4 * CUT_TOLERANCE[dtype] if dtype == "float32" else CUT_TOLERANCE[dtype]     # (float sums in another order, over 90 keys and 3 layers)
    for name in ("recorded", "plain"):
        assert float(((outputs[name] - outputs["apart"]).abs() / scale).max()) <= tolerance
    assert torch.isfinite(outputs["recorded"]).all()


def test_recordings_of_changing_groups(tmp_path, always_shared):
    """One recording serves steps whose groups come and go; rows in no group beside them."""
    folder = make_model(tmp_path / "m", CONFIG_A, 7, "float32")
    engines = [Engine(folder, dtype="float32", max_tokens=4096, max_requests=16, capture_graphs=capture) for capture in (True, False)]
    one, two = random_tokens(5, 60, 256), random_tokens(6, 33, 256)
    for engine in engines:
        for name, prompt in (("a0", one), ("b0", two), ("alone", random_tokens(7, 50, 256))):
            engine.admit(name)
            engine.step([StepEntry(name, prompt, [])])
        for index in range(1, 4):
            engine.cache.fork("a0", f"a{index}", 59)
            engine.cache.fork("b0", f"b{index}", 32)
    steps = [["a1", "a2", "a3", "alone", "b1", "b2"], ["a0", "a1", "a2", "b0", "b3", "b1"], ["alone", "a1", "a3", "b1", "b3", "a2"],
             ["a0", "alone", "b0", "b1", "a2", "a3"], ["a1", "a2", "a3", "alone", "b1", "b2"]]
    for turn, names in enumerate(steps):
        entries = [StepEntry(name, [(13 * turn + place) % 256], [0]) for place, name in enumerate(names)]
        recorded, laid_out = [engine.step(entries) for engine in engines]
        assert torch.equal(recorded, laid_out), turn
    for engine in engines:
        engine.cache.check()


def test_where_it_pays_it_is_done_by_itself(tmp_path, counted):
    folder = make_model(tmp_path / "m", CONFIG_WIDE, 8, "bfloat16")
    engine = Engine(folder, dtype="bfloat16", max_tokens=8192, max_requests=16)
    out = engine.generate([random_tokens(8, 640, 256)], answers=8, max_tokens=4, temperature=1.0, top_k=50, min_p=0.01, seed=3)
    assert len(out) == 1 and [len(answer) for answer in out[0]] == [4] * 8 and counted
    counted.clear()
    engine.generate([random_tokens(9, 64, 256)], answers=8, max_tokens=4, temperature=1.0, seed=3)
    assert not counted                                    # too short to pay


def test_filters_and_log_probabilities(tmp_path):
    folder = make_model(tmp_path / "m", CONFIG_A, 9, "float32", std=0.3)
    engine = Engine(folder, dtype="float32", max_tokens=2048, max_requests=8)
    prompts = [random_tokens(10 + i, 9 + 5 * i, 256) for i in range(5)]
    greedy = engine.generate(prompts, max_tokens=10)
    assert engine.generate(prompts, max_tokens=10, temperature=1.3, top_k=1, seed=2) == greedy
    assert engine.generate(prompts, max_tokens=10, temperature=1.3, min_p=1.0, seed=2) == greedy
    for options in (dict(), dict(temperature=0.8, top_p=0.9, seed=4), dict(temperature=1.1, top_k=12, min_p=0.02, top_p=0.9, seed=4)):
        logprobs = []
        with_them = engine.generate(prompts, max_tokens=8, logprobs=logprobs, **options)
        assert with_them == engine.generate(prompts, max_tokens=8, **options)
        for prompt, tokens, values in zip(prompts, with_them, logprobs):
            assert len(values) == len(tokens)
            engine.admit("check")
            logits = engine.step([StepEntry("check", prompt + tokens[:-1], list(range(len(prompt) - 1, len(prompt) + len(tokens) - 1)))])
            engine.finish("check")
            want = torch.log_softmax(logits.double().cpu(), dim=-1)[torch.arange(len(tokens)), torch.tensor(tokens)]
            # logits of another cut of the same request: 1e-6 of the largest of a row each (see CUT_TOLERANCE), rounding beside them
            bound = 2 * CUT_TOLERANCE["float32"] * float(logits.abs().max()) + 2.0 ** -20
            assert float((torch.tensor(values, dtype=torch.float64) - want).abs().max()) <= bound


def test_a_rows_draw_does_not_depend_on_the_step_it_is_in():
    from tlie_amd.sampling.sampler import Sampler
    gen = torch.Generator().manual_seed(1)
    logits = (2.0 * torch.randn((6, 900), generator=gen)).to(DEV)
    params = [SamplingParams(temperature=0.0), SamplingParams(temperature=0.9, top_p=0.8, seed=5), SamplingParams(temperature=0.9, top_k=20, seed=5),
              SamplingParams(temperature=1.2, min_p=0.05, seed=9, logprobs=True), SamplingParams(temperature=1.0, seed=1), SamplingParams(logprobs=True)]
    sampler = Sampler(DEV, capacity=8)
    counters = [3, 1, 4, 1, 5, 9]
    together = sampler.sample_async(logits, params, counters)
    tokens, logprobs = together.read(), together.read_logprobs()
    want = torch.log_softmax(logits.double().cpu(), dim=-1)
    for row in range(6):
        alone = sampler.sample_async(logits[row:row + 1].contiguous(), [params[row]], [counters[row]])
        assert alone.read() == [tokens[row]]
        assert abs(logprobs[row] - float(want[row, tokens[row]])) <= 2.0 ** -19
        assert (alone.read_logprobs() is None) == (not params[row].logprobs)
    bad = logits.clone()
    bad[2, 5] = math.nan
    from tlie_amd.errors import EngineError
    with pytest.raises(EngineError):
        sampler.sample(bad, params, counters)


def test_answers_that_outnumber_the_pool(tmp_path, always_shared):
    """Preempted and recomputed, the tokens stay what they are."""
    folder = make_model(tmp_path / "m", CONFIG_A, 12, "float32")
    prompts = [random_tokens(20, 40, 256), random_tokens(21, 30, 256)]
    options = dict(max_tokens=30, temperature=0.8, seed=1, answers=5)
    ample = Engine(folder, dtype="float32", max_tokens=4096, max_requests=16)
    tight = Engine(folder, dtype="float32", max_tokens=192, max_requests=16)
    stats = {}
    want = ample.generate(prompts, **options)
    assert tight.generate(prompts, stats=stats, admit_partial=True, **options) == want
    assert stats["preemptions"] > 0 and tight.cache.free_pages() == [tight.cache.num_pages]


def test_the_command_line(tmp_path, capsys):
    from tlie_amd.cli import main
    folder = make_model(tmp_path / "m", CONFIG_A, 13, "float32")
    text = "ids:" + ",".join(str(token) for token in random_tokens(30, 40, 256))
    arguments = ["generate", folder, text, "6", "--dtype", "float32", "--temperature", "0.9", "--top-k", "30", "--min-p", "0.01", "--answers", "3", "--logprobs"]
    assert main(arguments) == 0
    out = json.loads(capsys.readouterr().out)
    assert len(out["answers"]) == 3 and out["answers"][0] == out["generated_tokens"] and all(len(answer) == 6 for answer in out["answers"])
    assert [len(values) for values in out["answer_logprobs"]] == [6, 6, 6] and out["logprobs"] == out["answer_logprobs"][0]
    for wrong in (["--answers", "0"], ["--top-k", "-2"], ["--min-p", "1.5"]):
        assert main(["generate", folder, text, "6", "--dtype", "float32", "--temperature", "0.9", *wrong]) != 0
        capsys.readouterr()


@pytest.mark.parametrize("filters", [dict(top_k=20), dict(min_p=0.05), dict(logprobs=True), dict(top_k=20, logprobs=True), dict()])
def test_logits_that_are_not_finite_are_errors_whatever_the_draw(filters):
    """An infinity of either sign or a NaN: `numerical_error`, for rows with filters as for rows without."""
    from tlie_amd.errors import EngineError
    from tlie_amd.sampling.sampler import Sampler
    sampler = Sampler(DEV, capacity=4)
    params = [SamplingParams(temperature=0.8, seed=index, **filters) for index in range(3)]
    logits = torch.randn((3, 700), generator=torch.Generator().manual_seed(2)).to(DEV)
    assert len(sampler.sample(logits, params, [0, 0, 0])) == 3
    for value in (-math.inf, math.inf, math.nan):
        bad = logits.clone()
        bad[1, 33] = value
        with pytest.raises(EngineError):
            sampler.sample(bad, params, [0, 0, 0])


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_steps_that_mix_a_family_with_portions_are_recorded(tmp_path, dtype, always_shared, counted):
    """Answers that decode beside portions of other prompts, and portions of the family's own: by one recording per size, with changing
    cuts, the same as launched one by one on its arrays; and, up to the other order of sums, as unrecorded and as the ordinary attention has it."""
    folder = make_model(tmp_path / "m", CONFIG_B, 14, dtype)
    prompt = random_tokens(40, 90, 512)
    steps = [[("a", 1), ("b", 1), ("c", 1), ("x", 9)], [("x", 7), ("a", 1), ("b", 1)], [("a", 1), ("b", 1), ("c", 1), ("x", 9)],
             [("b", 5), ("c", 3), ("x", 1), ("a", 1)], [("x", 2), ("y", 9), ("a", 1), ("c", 1)], [("a", 2), ("b", 2), ("c", 2), ("y", 1)]]
    outputs = {}
    for name, options in (("recorded", {}), ("laid out", dict(capture_graphs=False)), ("plain", dict(use_graphs=False)), ("ordinary", dict(use_graphs=False))):
        engine = Engine(folder, dtype=dtype, max_tokens=4096, max_requests=8, **options)
        if name == "ordinary":
            engine.runner.shared_groups = lambda entries: []
        for request in "axy":
            engine.admit(request)
        engine.step([StepEntry("a", prompt, [])])
        for request in "bc":
            engine.cache.fork("a", request, 85)
            engine.step([StepEntry(request, prompt[85:], [])])
        counted.clear()
        others = len(engine.runner._portion_graphs)           # (of the prompts)
        logits, at = [], 0
        for step in steps:
            entries = []
            for request, count in step:
                entries.append(StepEntry(request, [(31 * at + 7 * place) % 512 for place in range(count)], [count - 1]))
                at += count
            logits.append(engine.step(entries))
        if name == "recorded":
            assert len(engine.runner._shared_portion_graphs) == 1 and len(engine.runner._portion_graphs) == others
            assert len(counted) == 2 * 3                      # each layer twice, to run and to record; the other steps are replays
        else:
            assert len(counted) == (0 if name == "ordinary" else 3 * len(steps))
        engine.cache.check()
        outputs[name] = torch.cat(logits).double().cpu()
    assert torch.equal(outputs["recorded"], outputs["laid out"])
    scale = outputs["ordinary"].abs().amax(dim=-1, keepdim=True)
    # two results of different cuts, each within the bound of the truth (float: as above, over 3 layers)
    tolerance = 4 * CUT_TOLERANCE[dtype] if dtype == "float32" else CUT_TOLERANCE[dtype]
    for name in ("recorded", "plain"):
        assert float(((outputs[name] - outputs["ordinary"]).abs() / scale).max()) <= tolerance
