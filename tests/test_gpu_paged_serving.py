"""GPU: the serving example (examples/paged_serving.py) end to end.

Two ways through the same layers differ by their bf16 roundings alone: about six
to a layer, 2^-9 of a value each, which four layers can add up to 24 x 2^-9 of the
largest logit: 2^-4.
"""
import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example():
    path = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "examples", "paged_serving.py")
    spec = importlib.util.spec_from_file_location("paged_serving", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def tokens(n, seed):
    return torch.randint(2048, (n,), generator=torch.Generator().manual_seed(seed)).tolist()


def close(a, b):
    return float((a.float() - b.float()).abs().max()) <= 2.0 ** -4 * float(b.float().abs().max())


def test_main(example, dev, capsys):
    example.main(["--steps", "3"])
    example.main(["--steps", "3", "--bits", "4"])
    assert "pages in use" in capsys.readouterr().out


def test_chunks_and_company_do_not_matter(example, dev):
    """A prompt in one piece and alone, or in chunks beside other sequences."""
    alone, served = example.Server(), example.Server()
    prompt, other = tokens(150, 1), tokens(90, 2)
    want = alone.step([0], [prompt])
    served.step([5, 2], [prompt[:70], other[:1]])
    served.step([2, 5], [other[1:], prompt[70:149]])
    got = served.step([2, 5], [[3], prompt[149:]])[1:]
    assert close(got, want)
    alone.check()
    served.check()


def test_a_fork_goes_on_like_its_parent(example, dev):
    server = example.Server()
    server.step([0], [tokens(150, 1)])
    server.fork([0, 0], [1, 2])
    logits = server.step([0, 1, 2], [[7], [7], [8]])
    assert close(logits[1:2], logits[0:1])
    assert not close(logits[2:3], logits[0:1])
    server.check()


@pytest.mark.parametrize("bits", [16, 4])
def test_freeing_trimming_and_compaction_change_no_result(example, dev, bits):
    a, b = example.Server(bits=bits), example.Server(bits=bits)
    for s in (a, b):
        s.step([0, 1, 2], [tokens(100, 3), tokens(150, 4), tokens(5, 5)])
    b.release(free=[0], trim=[1, 2])
    before = {kind: int((c.refs > 0).sum()) for kind, c in b.caches.items()}
    assert b.compact() == before
    assert before["sliding"] < before["full"]  # the window's pages alone
    for kind, n in before.items():
        assert int((b.caches[kind].refs[:n] > 0).sum()) == n
    ids = [tokens(9, 6), tokens(1, 7)]
    assert torch.equal(a.step([1, 2], ids), b.step([1, 2], ids))
    a.check()
    b.check()
