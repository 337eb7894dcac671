"""``generate`` with beams and with a common prefix: what it prints, and the options that exclude one another."""
import json

import pytest

from conftest import prompts_for
from test_cli import run


def printed(p):
    assert p.returncode == 0, p.stderr
    return [json.loads(line) for line in p.stdout.splitlines() if line.strip()]


def ids(prompts):
    return ";".join(",".join(str(t) for t in p) for p in prompts)


@pytest.mark.gpu
def test_beams_print_what_the_search_finds(folders):
    from quicknn_b200.engine import LLM
    from quicknn_b200.sampling import BeamOptions
    folder, prompts = folders("A", "float32"), prompts_for("A", [5, 11])
    llm = LLM(folder, max_context=64, dtype="float32")
    stop = llm.beam_search(prompts[:1], BeamOptions(beams=1, max_new_tokens=4), stop_ids=[])[0].replies[0].tokens[3]
    want = llm.beam_search(prompts, BeamOptions(beams=3, max_new_tokens=6, length_penalty=0.7, replies=2), stop_ids=[stop])
    got = printed(run("generate", "--model", folder, "--prompt-ids", ids(prompts), "--max-new-tokens", "6", "--dtype", "float32", "--max-context", "64",
                      "--stop-ids", str(stop), "--beams", "3", "--replies", "2", "--length-penalty", "0.7", "--profile"))
    assert [g["request"] for g in got] == [0, 1] and [g["prompt_tokens"] for g in got] == [5, 11]
    for g, w in zip(got, want):
        assert [r["tokens"] for r in g["replies"]] == [r.tokens for r in w.replies] and len(w.replies) == 2
        assert [r["finish_reason"] for r in g["replies"]] == [r.finish_reason for r in w.replies]
        assert all(abs(r["score"] - v.score) <= 1e-5 * max(1, abs(v.score)) for r, v in zip(g["replies"], w.replies))


@pytest.mark.gpu
def test_a_common_prefix(folders, plain_models):
    folder, plain = folders("A", "float32"), plain_models("A", "float32")
    prefix, *prompts = prompts_for("A", [20, 3, 6])
    got = printed(run("generate", "--model", folder, "--prompt-ids", ids(prompts), "--prefix-ids", ids([prefix]), "--max-new-tokens", "5",
                      "--temperature", "0", "--dtype", "float32", "--max-context", "64", "--stop-ids", ""))
    for g, p in zip(got, prompts):
        assert g["tokens"] == plain.greedy(prefix + p, 5) and g["prompt_tokens"] == 20 + len(p) and g["reused_tokens"] == 20


@pytest.mark.gpu
def test_options_that_exclude_one_another(folders):
    folder = folders("A", "float32")
    for extra in (["--beams", "2", "--turns"], ["--beams", "2", "--stream"], ["--beams", "2", "--prefix-ids", "5"], ["--turns", "--prefix-ids", "5"],
                  ["--beams", "2", "--replies", "3"], ["--beams", "-1"], ["--beams", "2", "--length-penalty", "nan"]):
        p = run("generate", "--model", folder, "--prompt-ids", "5", *extra)
        assert p.returncode not in (0, 3), extra
