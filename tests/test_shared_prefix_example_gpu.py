"""The example that decodes several answers from one prompt over a 4-bit cache with shared pages: the
answers are those of sequences that each hold their own copy of the prompt, pages are shared, and
decoding goes on after freeing and compacting."""
import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_spec = importlib.util.spec_from_file_location("shared_prefix_q4", os.path.join(ROOT, "examples", "shared_prefix_q4.py"))
E = importlib.util.module_from_spec(_spec)
_spec.loader.exec_module(E)


@pytest.mark.parametrize("n_prompt", [1, 64, 131])
def test_forked_answers_match_separate_prompts(n_prompt):
    prompt = [(7 * i * i + 3) % E.CONFIG["vocab"] for i in range(n_prompt)]
    n, tokens = 5, 12
    runs = []
    for share in (True, False):
        dec = E.Decoder(n_seq=n, max_seq=n_prompt + tokens + 2, n_pages=48)
        got, logits = E.answers(dec, prompt, n, tokens, share)
        assert dec.status.item() == 0
        runs.append((dec, got, torch.stack(logits)))
    (dec, got, lg), (other, want, lw) = runs
    # the same kernels on the same inputs, split over the warps alike: the caches agree bit for bit
    assert got == want
    assert torch.equal(lg, lw)
    whole = n_prompt // dec.page
    total = -(-(n_prompt + tokens - 1) // dec.page)
    assert other.pages_in_use() == n * total
    assert dec.pages_in_use() == whole + n * (total - whole)
    # free some, compact, and go on: both caches still hold the same
    for d in (dec, other):
        d.free([0, 3])
        in_use, _ = d.compact()
        assert in_use == d.pages_in_use() == int(d.ref[:in_use].count_nonzero())
    left = [1, 2, 4]
    a, b = (d.step([got[s][-1] for s in left], left) for d in (dec, other))
    assert torch.equal(a, b) and dec.status.item() == 0 and other.status.item() == 0


def test_example_runs(capsys):
    E.main(["--prompt", "70", "--answers", "3", "--tokens", "4"])
    out = capsys.readouterr().out
    assert "pages in use" in out and "next tokens" in out


@pytest.mark.parametrize("prompt,n,tokens", [(70, 1, 3), (5, 1, 1), (130, 37, 3), (4600, 2, 2), (64, 3, 130)])
def test_example_takes_any_size(capsys, prompt, n, tokens):
    """One answer, more answers than rows of a pass, prompts and answers of many pages."""
    E.main(["--prompt", str(prompt), "--answers", str(n), "--tokens", str(tokens)])
    lines = capsys.readouterr().out.splitlines()
    assert [x.split(":")[0] for x in lines[:n]] == ["answer %d" % i for i in range(n)]
    assert ("next tokens" in lines[-1]) == (n > 1)


def test_steps_in_groups_are_those_of_each_group():
    prompt = [(5 * i + 1) % E.CONFIG["vocab"] for i in range(70)]
    n = E.CHUNK + 3
    decs = [E.Decoder(n_seq=n, max_seq=90, n_pages=48) for _ in range(2)]
    ids = [(11 * i) % E.CONFIG["vocab"] for i in range(n)]
    for d in decs:
        d.prompt(prompt, 0)
        d.fork(0, list(range(1, n)))
    whole = decs[0].step(ids, list(range(n)))
    parts = [decs[1].step(ids[a:b], list(range(a, b))) for a, b in ((0, E.CHUNK), (E.CHUNK, n))]
    assert torch.equal(whole, torch.cat(parts))
    for d in decs:
        d.check()


@pytest.mark.parametrize("args", [["--answers", "0"], ["--prompt", "0"], ["--tokens", "0"], ["--answers", "5000"]])
def test_example_refuses_sizes_that_are_none(capsys, args):
    with pytest.raises(SystemExit):
        E.main(args)
    assert "at least 1" in capsys.readouterr().err


def test_a_pool_that_runs_out_is_reported():
    dec = E.Decoder(n_seq=2, max_seq=256, n_pages=2)
    dec.prompt(list(range(200)), 0)
    with pytest.raises(RuntimeError):
        dec.check()
