"""The documented example of the 8-bit row operators, run as it stands: what it calls neighbours are the rows'
neighbours, also where the rows' sizes differ widely."""
import re
from pathlib import Path

import numpy as np
import pytest
import torch

from tests import int8_oracle as R

ROOT = Path(__file__).resolve().parent.parent


def example():
    section = (ROOT / "INTEGRATION.md").read_text().split("## 8.")[1]
    return re.search(r"```python\n(.*?)```", section, re.S).group(1)


def data():
    """2,000 rows of 96 whose sizes span a factor of 20, and 50 queries."""
    g = np.random.default_rng(11)
    rows = g.standard_normal((2000, 96)) * np.exp(g.uniform(0, 3, (2000, 1)))
    return rows.astype(np.float32), g.standard_normal((50, 96)).astype(np.float32)


def best(scores, k=10):
    return np.argsort(-scores, axis=1, kind="stable")[:, :k]


def recall(found, want):
    return np.mean([len(set(a.tolist()) & set(b.tolist())) for a, b in zip(found, want)]) / want.shape[1]


def test_what_the_scales_are_for():
    """On the CPU, from the definitions: scaled products and codes of one scale keep the order of these rows, codes of a
    scale each do not."""
    rows, queries = data()
    want = best(queries.astype(np.float64) @ rows.T.astype(np.float64))
    (q, sq), (c, sc) = R.quantize(queries), R.quantize(rows)
    one = np.rint(rows / (np.abs(rows).max() / 127))
    assert recall(best(R.gemm(q, c, sq, sc)), want) > 0.9
    assert recall(best(q.astype(np.float64) @ one.T), want) > 0.9
    assert recall(best(q.astype(np.float64) @ c.T.astype(np.float64)), want) < 0.5


@pytest.mark.gpu
def test_example():
    rows, queries = data()
    g = torch.Generator(device="cuda").manual_seed(2)
    rand = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    held, heads, dim, pages, page_size = 40, 2, 64, 4, 16
    names = {"torch": torch, "weight": rand(48, 96), "x": rand(5, 96), "bias": rand(48),
             "embeddings": torch.from_numpy(rows).cuda(), "queries": torch.from_numpy(queries).cuda(),
             "pages": pages, "page_size": page_size, "heads": heads, "dim": dim,
             "keys": rand(held, heads, dim), "values": rand(held, heads, dim),
             "slots": torch.arange(held, device="cuda"), "page_table": torch.arange(pages, device="cuda")[None].int(),
             "offsets": torch.tensor([0, held], device="cuda"), "total": held}
    given = dict(names)
    exec(example(), names)
    want = queries.astype(np.float64) @ rows.T.astype(np.float64)
    (q, sq), (c, sc) = R.quantize(queries), R.quantize(rows)
    scaled = R.gemm(q, c, sq, sc)
    found = names["neighbours"].cpu().numpy()
    # the scores are within their roundings of the definition's, so the best are the best to within them
    bound = 2 * R.gemm_bound(scaled, None, 2.0 ** -23).max(1, keepdims=True)
    top = np.sort(scaled, axis=1)[:, ::-1][:, :10]
    assert (np.abs(np.take_along_axis(scaled, found, 1) - top) <= bound).all()
    assert recall(found, best(want)) > 0.9
    assert recall(names["rows"].cpu().numpy(), best(want)) > 0.9
    # one step of a row's or channel's codes is off by half a scale
    full = (given["x"].double() @ given["weight"].double().t() + given["bias"].double())
    step = lambda t: t.double().abs().amax(1) / 127 / 2  # noqa: E731
    x1, w1 = (t.double().abs().sum(1) for t in (given["x"], given["weight"]))
    off = step(given["x"])[:, None] * w1 + x1[:, None] * step(given["weight"]) + 96 * step(given["x"])[:, None] * step(given["weight"])
    assert ((names["y"].double() - full).abs() <= off * 1.001 + full.abs() * 2.0 ** -20).all()
    for name in ("keys", "values"):
        x, got = given[name].double(), names[name].double()
        assert ((got - x).abs() <= x.abs().amax(-1, keepdim=True) / 127 / 2 * 1.001 + x.abs() * 2.0 ** -7).all()
