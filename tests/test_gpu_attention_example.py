"""examples/embed_and_search.py: documents, queries over a forked prefix, the scan and the reader together."""
import importlib.util
import os

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("embed_and_search", os.path.join(ROOT, "examples", "embed_and_search.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def test_example_runs(example):
    r = example.main()
    assert r["status"] == 0
    assert r["lens"][0] == 150
    assert r["lens"][1:6] == [150 + q + d + 70 for q, d in zip(r["query_lens"], r["doc_lens"])]
    assert all(0 <= b < 640 for b in r["best"])
    # the scan's first hit is near the best exact inner product
    dots = r["q_emb"] @ r["emb"].T
    assert all(dots[i, b] >= np.sort(dots[i])[-40] for i, b in enumerate(r["best"]))
    assert r["answers"].shape == (70, 5) and 0 <= r["answers"].min() and r["answers"].max() < 1000
    assert r["compacted"] < r["trimmed"] <= r["held"]
    again = example.main()
    assert again["best"] == r["best"] and np.array_equal(again["answers"], r["answers"]) and again["again"] == r["again"]


def test_cached_and_packed_passes_agree(example):
    """The same tokens through `window_attention` and through the cache (an instruction, a fork, the rest): the
    pooled embeddings agree as far as keys and values in 8 bits allow (relative rounding 2^-8 per value, two
    layers of averages: well under 2% of a unit vector)."""
    import mrl_b200 as M

    dev = M.Device(0)
    dev.use_torch_stream()
    model = example.Model()
    rng = np.random.default_rng(3)
    text = rng.integers(0, example.VOCAB, 300)
    whole = example.embed_documents(model, dev, [text])
    reader = example.Reader(model, dev)
    a, _ = reader.extend([0], [text[:150]])
    reader.cache.fork(example.i32([0]), example.i32([3]))
    b, _ = reader.extend([3], [text[150:]])
    e = np.concatenate([a.float().cpu().numpy(), b.float().cpu().numpy()]).mean(0)
    e /= np.linalg.norm(e)
    assert np.linalg.norm(e - whole[0]) < 0.02
    dev.close()
