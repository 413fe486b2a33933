"""Tensors that the search entry points take as bare addresses: those that are no [n, dimension] rows of the index's
type on a CUDA device are refused, and views whose rows do not follow one another are read as the rows they show."""
import numpy as np
import pytest
import torch

from elips_b200 import DimensionMismatch
from elips_b200.exact import ExactIndex
from elips_b200.ivfpq import IvfFlatIndex, IvfPqIndex
from elips_b200.quant import QuantizedIndex


def bare(kind, **attributes):
    """An index without its device half: the checks come before it is touched."""
    ix = kind.__new__(kind)
    ix.__dict__.update(dimension=8, device=0, _h=None, **attributes)
    return ix


ENTRIES = {
    "exact add": lambda x: bare(ExactIndex, precision="fp32").add_device(x),
    "exact": lambda x: bare(ExactIndex, precision="fp32").search_device(x, 1),
    "exact candidates": lambda x: bare(ExactIndex, precision="fp32").search_candidates_device(x, 1, 0, None),
    "exact shared": lambda x: bare(ExactIndex, precision="fp32").search_candidates_shared_device(x, 1, 0, None, None),
    "pq add": lambda x: bare(IvfPqIndex).add_device(x, torch.zeros(4, dtype=torch.int32)),
    "pq probe": lambda x: bare(IvfPqIndex, nprobe=1, n_lists=1).probe_device(x),
    "pq candidates": lambda x: bare(IvfPqIndex).search_candidates_device(x, 1),
    "pq rerank": lambda x: bare(IvfPqIndex).rerank_device(x, 1, None),
    "pq": lambda x: bare(IvfPqIndex).search_device(x, 1),
    "flat add": lambda x: bare(IvfFlatIndex).add_device(x, torch.zeros(4, dtype=torch.int32)),
    "flat": lambda x: bare(IvfFlatIndex).search_device(x, 1),
    "quantized": lambda x: bare(QuantizedIndex).search_device(x, 1),
}


@pytest.mark.parametrize("entry", ENTRIES)
def test_refused(entry):
    call = ENTRIES[entry]
    for x in (torch.zeros(8), torch.zeros((4, 7)), torch.zeros((2, 4, 8))):
        with pytest.raises(DimensionMismatch):
            call(x)
    for x in (torch.zeros((4, 8), dtype=torch.float16), torch.zeros((4, 8), dtype=torch.float64),
              torch.zeros((4, 8), dtype=torch.int8), torch.zeros((4, 8))):           # the last: not on a CUDA device
        with pytest.raises(ValueError):
            call(x)


def test_int8_index_takes_codes():
    with pytest.raises(ValueError, match="int8"):
        bare(ExactIndex, precision="int8").search_device(torch.zeros((4, 8)), 1)
    with pytest.raises(ValueError, match="CUDA"):
        bare(ExactIndex, precision="int8").search_device(torch.zeros((4, 8), dtype=torch.int8), 1)


def test_rows_on_another_device():
    """A tensor of cuda:1 for an index on cuda:0 (a stand-in: this needs no GPU)."""
    class Elsewhere:
        shape, dtype, is_cuda, device = (4, 8), torch.float32, True, "cuda:1"
        dim, get_device = (lambda self: 2), (lambda self: 1)
    with pytest.raises(ValueError, match="cuda:0"):
        bare(ExactIndex, precision="fp32").search_device(Elsewhere(), 1)
    with pytest.raises(ValueError, match="cuda:0"):
        bare(IvfFlatIndex).search_device(Elsewhere(), 1)


def views(x):
    """Tensors of other strides, each with the rows it shows."""
    n, d = x.shape
    wide = torch.full((n, d + 13), float("nan") if x.is_floating_point() else 77, dtype=x.dtype, device=x.device)
    wide[:, 5:5 + d] = x
    every = torch.full((3 * n, d), 77, dtype=x.dtype, device=x.device)
    every[::3] = x
    return {"slice": (wide[:, 5:5 + d], x), "step": (every[::3], x), "transposed": (x.t().contiguous().t(), x),
            "broadcast": (x[2].expand(n, d), x[2].repeat(n, 1))}


@pytest.mark.gpu
@pytest.mark.parametrize("view", ["slice", "step", "transposed", "broadcast"])
@pytest.mark.parametrize("precision,metric", [("fp32", "euclidean"), ("int8", "dot_product")])
def test_exact_search_of_views(precision, metric, view):
    g = torch.Generator(device="cuda").manual_seed(3)
    base, q = torch.randn((3000, 100), generator=g, device="cuda"), torch.randn((37, 100), generator=g, device="cuda")
    if precision == "int8":
        base, q = ((t * 40).round().clamp(-127, 127).to(torch.int8) for t in (base, q))
    ix = ExactIndex(metric, 100, precision=precision)
    ix.add_device(views(base)["slice"][0])
    shown, rows = views(q)[view]
    want = ix.search_batch(rows.cpu().numpy(), 5)
    for got in (ix.search_device(shown, 5), ix.search_device(shown, 5, stream=0)):
        torch.cuda.synchronize()
        assert np.array_equal(got[0].cpu().numpy(), want[0]) and np.array_equal(got[1].cpu().numpy(), want[1])
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    got = ix.search_device(shown, 5, stream=s.cuda_stream)
    s.synchronize()
    assert np.array_equal(got[1].cpu().numpy(), want[1])
    cand = [torch.empty((37, 5, 2), dtype=torch.int32, device="cuda") for _ in range(2)]
    ix.search_candidates_device(shown, 5, 0, cand[0])
    ix.search_candidates_device(rows.contiguous(), 5, 0, cand[1])
    assert torch.equal(*cand)


@pytest.mark.gpu
@pytest.mark.parametrize("d", [100, 128])
def test_queries_as_quantize_rows_gives_them(d):
    """Codes are a view of wider rows where d is no multiple of 16."""
    from elips_b200 import int8
    g = torch.Generator(device="cuda").manual_seed(d)
    codes, _ = int8.quantize_rows(torch.randn((500, d), generator=g, device="cuda"))
    q, _ = int8.quantize_rows(torch.randn((40, d), generator=g, device="cuda"))
    ix = ExactIndex("dot_product", d, precision="int8")
    ix.add_device(codes)
    dist, rows = ix.search_device(q, 500)
    scores = q.cpu().double() @ codes.cpu().double().t()
    assert torch.equal(-dist.cpu().double(), scores.gather(1, rows.cpu()))
    assert torch.equal(-dist.cpu().double(), scores.sort(1, descending=True).values)


@pytest.mark.gpu
@pytest.mark.parametrize("view", ["slice", "transposed"])
def test_other_indexes_search_views(view):
    g = np.random.default_rng(4)
    base, q = g.standard_normal((2000, 32)).astype(np.float32), g.standard_normal((21, 32)).astype(np.float32)
    cent = base[:8].copy()
    asg = ((base[:, None] - cent) ** 2).sum(-1).argmin(1).astype(np.uint32)
    book = g.standard_normal((4, 256, 8)).astype(np.float32)
    flat = IvfFlatIndex("euclidean", 32, cent, 3)
    pq = IvfPqIndex("euclidean", 32, cent, book, nprobe=3)
    shown_base = views(torch.from_numpy(base).cuda())[view][0]
    lists = torch.from_numpy(asg.view(np.int32)).cuda()
    flat.add_device(shown_base, lists)
    pq.add_device(shown_base, lists)
    shown = views(torch.from_numpy(q).cuda())[view][0]
    plain = shown.contiguous()
    for ix in (flat, pq):
        assert all(torch.equal(a, b) for a, b in zip(ix.search_device(shown, 5), ix.search_device(plain, 5)))
    d, r = ix.search_batch(q, 5)
    assert np.array_equal(pq.search_device(shown, 5)[1].cpu().numpy(), r)
    assert torch.equal(pq.probe_device(shown), pq.probe_device(plain))
    cand = pq.search_candidates_device(shown, 5)
    assert torch.equal(cand, pq.search_candidates_device(plain, 5))
    assert all(torch.equal(a, b) for a, b in zip(pq.rerank_device(shown, 5, cand), pq.rerank_device(plain, 5, cand)))
