"""The command line's output for several prompts, answers and log-probabilities, with an engine that answers on the host."""
import json

import pytest

from tlie_amd import cli


class Answering:
    """Token p * 100 + a * 10 + i for prompt p, answer a, place i; its log-probability the negative of that."""

    def __init__(self, *args, **named):
        self.asked = named

    def generate(self, prompts, max_tokens, answers, logprobs, **options):
        tokens = [[[p * 100 + a * 10 + i for i in range(max_tokens)] for a in range(answers)] for p in range(len(prompts))]
        if answers == 1:
            tokens = [row[0] for row in tokens]
        if logprobs is not None:
            negated = lambda value: [negated(one) for one in value] if isinstance(value, list) else -float(value)
            logprobs[:] = negated(tokens)
        return tokens


@pytest.mark.parametrize("prompts", [1, 2, 3])
@pytest.mark.parametrize("answers", [1, 2, 4])
@pytest.mark.parametrize("logprobs", [False, True])
def test_every_answers_log_probabilities_are_printed(monkeypatch, capsys, prompts, answers, logprobs):
    monkeypatch.setattr(cli, "_engine", lambda args, positions, requests=1: Answering())
    text = ";".join("ids:" + ",".join(str(5 + token) for token in range(prompt + 3)) for prompt in range(prompts))
    assert cli.main(["generate", "nowhere", text, "3", "--answers", str(answers), *(["--logprobs"] if logprobs else [])]) == 0
    out = json.loads(capsys.readouterr().out)
    rows = out["requests"] if prompts > 1 else [out]
    assert len(rows) == prompts
    for p, row in enumerate(rows):
        tokens = [[p * 100 + a * 10 + i for i in range(3)] for a in range(answers)]
        values = [[-float(token) for token in answer] for answer in tokens]
        assert row["generated_tokens"] == tokens[0]
        assert ("answers" in row) == (answers > 1) and (answers == 1 or row["answers"] == tokens)
        assert ("logprobs" in row) == logprobs and (not logprobs or row["logprobs"] == values[0])
        assert ("answer_logprobs" in row) == (logprobs and answers > 1)
        assert "answer_logprobs" not in row or row["answer_logprobs"] == values
