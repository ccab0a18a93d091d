"""The router and the grouping of rows: every value against a plain 64-bit restatement, ties, masks and sizes at which the
kernels change their form."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def grouping_ref(ids, groups):
    """Stable grouping in plain Python order: (order, position, offsets)."""
    key = torch.where((ids < 0) | (ids >= groups), torch.full_like(ids, groups), ids).long().cpu()
    order = torch.argsort(key, stable=True)
    position = torch.empty_like(order)
    position[order] = torch.arange(order.numel())
    counts = torch.bincount(key, minlength=groups + 1)[:groups]
    return order, position, torch.cat([torch.zeros(1, dtype=torch.long), counts.cumsum(0)])


def check_grouping(g, ids, groups):
    for got, want in zip(g, grouping_ref(ids, groups)):
        assert got.dtype == torch.int32 and torch.equal(got.cpu().long(), want)


@pytest.mark.parametrize("rows,groups", [(0, 3), (1, 1), (1, 1024), (31, 2), (32, 2), (33, 7), (2048, 128), (2049, 128), (5000, 1),
                                         (8193, 1024), (16385, 60), (131072, 128), (300001, 1000)])
def test_group_rows(rows, groups):
    from llm_reproducibility_b200.tbik.row_groups import group_rows
    g = torch.Generator().manual_seed(rows + groups)
    ids = torch.randint(-2, groups + 2, (rows,), generator=g).to(torch.int32)  # some rows in no group
    check_grouping(group_rows(ids.cuda(), groups), ids, groups)


def test_group_rows_of_one_group_and_of_none():
    from llm_reproducibility_b200.tbik.row_groups import group_rows
    for value in (0, 4, -1, 5, 2 ** 31 - 1, -2 ** 31):
        ids = torch.full((777,), value, dtype=torch.int64).to(torch.int32)
        check_grouping(group_rows(ids.cuda(), 5), ids, 5)


def test_group_rows_takes_strided_ids_and_a_matrix():
    from llm_reproducibility_b200.tbik.row_groups import group_rows
    ids = torch.randint(0, 9, (40, 6), dtype=torch.int32)
    check_grouping(group_rows(ids.cuda()[:, ::2], 9), ids[:, ::2].reshape(-1), 9)


def route_ref(x, k, renormalize):
    """64-bit router: ids by (value, lower index first), weights by the softmax's definition, 0 for a row all -inf."""
    x = x.double().cpu()
    ids = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :k]
    top = x.gather(1, ids)
    over = top if renormalize else x
    peak = over.max(1, keepdim=True).values
    w = torch.exp(top - peak) / torch.exp(over - peak).sum(1, keepdim=True)
    return torch.where(peak == -math.inf, torch.zeros_like(w), w), ids


CASES = [(1, 1, 1), (1, 128, 8), (3, 2, 2), (5, 33, 32), (64, 64, 6), (512, 128, 8), (513, 128, 8), (777, 60, 4), (9, 257, 16),
         (40, 1024, 32), (2000, 512, 10), (4099, 8, 2),
         (0, 4, 2), (40, 1024, 8), (7, 300, 8), (5, 8, 8), (3, 5, 3), (2000, 16, 2), (64, 17, 5), (20000, 128, 8), (17000, 24, 1)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("T,E,k", CASES)
def test_route(T, E, k, renormalize, dtype):
    from llm_reproducibility_b200.tbik.row_groups import route_topk
    g = torch.Generator().manual_seed(T * 1000 + E + k)
    x = (torch.randn(T, E, generator=g) * 2).to(dtype)  # 16-bit scores: many exact ties
    r = route_topk(x.cuda(), k, renormalize=renormalize)
    w, ids = route_ref(x, k, renormalize)
    assert torch.equal(r.ids.cpu().long(), ids)
    check_grouping(r.groups, ids.flatten(), E)
    # exp is off by at most 2 units (2^-23 each) at either end, its argument's rounding by 2^-24 |x - peak| <= 2^-24 * 20,
    # the sum of up to E terms by E 2^-24 at the very most, the quotient by 2^-24
    tol = (4 + 20 + E) * 2.0 ** -23
    assert ((r.weights.cpu().double() - w).abs() <= tol * w + 1e-38).all()
    if renormalize and T:
        assert (r.weights.sum(1) - 1).abs().max() < tol


def test_route_of_masked_rows_infinities_and_nan():
    from llm_reproducibility_b200.tbik.row_groups import route_topk
    inf, nan = math.inf, math.nan
    x = torch.tensor([[-inf, -inf, -inf, -inf], [-inf, 1.0, -inf, -inf], [0.0, -0.0, 0.0, -0.0], [1.0, nan, 5.0, nan],
                      [torch.finfo(torch.float32).min] * 4, [2.0, inf, 1.0, 0.0], [-inf, 3.0, -inf, 2.0]])
    for renormalize in (True, False):
        r = route_topk(x.cuda(), 3, renormalize=renormalize)
        ids, w = r.ids.cpu().tolist(), r.weights.cpu()
        assert ids[0] == [0, 1, 2] and w[0].tolist() == [0.0, 0.0, 0.0]          # nothing left: no weight
        assert ids[1] == [1, 0, 2] and w[1].tolist() == [1.0, 0.0, 0.0]
        assert ids[2] == [0, 1, 2]                                              # -0 equals +0
        assert ids[3] == [1, 3, 2] and w[3].isnan().all()                       # NaN is not hidden
        assert ids[4] == [0, 1, 2] and torch.allclose(w[4], torch.full((3,), 1 / 3 if renormalize else 0.25), atol=1e-7)
        assert ids[5][0] == 1 and w[5].isnan().any()
        assert ids[6] == [1, 3, 0] and w[6][2] == 0.0
        check_grouping(r.groups, r.ids.flatten(), 4)


def hard_rows(E, dtype):
    """Rows of E scores at which a key can go wrong: masks, infinities, NaN of either sign, zeros of either sign, the type's lowest and
    smallest numbers, ties."""
    inf, nan, f = math.inf, math.nan, torch.finfo(dtype)
    g = torch.Generator().manual_seed(E)
    normal = torch.randn(E, generator=g)
    fill = lambda v: torch.full((E,), float(v))  # noqa: E731
    at = lambda row, v, *places: row.clone().index_fill_(0, torch.tensor([q % E for q in places]), float(v))  # noqa: E731
    rows = [fill(-inf), at(fill(-inf), 1.0, 1), at(fill(-inf), -3.0, E - 1, 0, 7), torch.tensor([0.0, -0.0]).repeat(E)[:E],
            torch.tensor([-0.0, 0.0, 0.0]).repeat(E)[:E], at(normal, nan, 1, 3), at(normal, nan, E - 1), fill(nan), at(fill(-inf), nan, 2),
            -at(normal, nan, 4), fill(f.min), at(fill(f.min), -inf, 0, 5, E - 1), at(fill(-inf), f.min, 3), at(normal, inf, 2), at(normal, inf, 0, E - 1),
            at(at(normal, inf, 3), -inf, 1), at(at(normal, inf, 1), nan, 2), at(normal, -inf, *range(0, E, 2)), at(normal, f.max, 0, 1),
            at(normal, f.min, 0, 1), torch.arange(E) * f.smallest_normal * f.eps - 3 * f.smallest_normal * f.eps, fill(f.smallest_normal * f.eps),
            at(fill(-f.smallest_normal * f.eps), 0.0, 2), (normal * 2).round(), fill(1.0)]
    return torch.stack(rows).to(dtype)


def hard_ref(x, k, renormalize):
    """Ids by (NaN first, then value, lower index first); weights by the definition, whose NaN are kept."""
    x = x.double()
    by_value = torch.sort(torch.where(x.isnan(), 0.0, x), dim=1, descending=True, stable=True).indices
    nan_first = torch.sort(x.isnan().gather(1, by_value).int(), dim=1, descending=True, stable=True).indices
    ids = by_value.gather(1, nan_first)[:, :k]
    top = x.gather(1, ids)
    over = top if renormalize else x
    peak = top[:, :1]
    w = torch.exp(top - peak) / torch.exp(over - peak).sum(1, keepdim=True)
    return torch.where(peak == -math.inf, torch.zeros_like(w), w), ids


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("E,k", [(9, 3), (8, 8), (128, 8), (127, 5), (300, 8), (1024, 8), (40, 9), (128, 32), (300, 16), (512, 12), (1000, 32)])
def test_route_of_hard_rows_in_every_form(E, k, renormalize, dtype):
    from llm_reproducibility_b200.tbik.autograd import tree_route_topk
    from llm_reproducibility_b200.tbik.row_groups import route_topk
    x = hard_rows(E, dtype)
    w, ids = hard_ref(x, k, renormalize)
    for times in (1, 700):  # one launch, and the form of many tokens
        r = route_topk(x.cuda().repeat(times, 1), k, renormalize=renormalize)
        got = r.weights.cpu().double()
        for part in (slice(0, len(x)), slice(-len(x), None)):
            assert torch.equal(r.ids[part].cpu().long(), ids)
            assert torch.equal(got[part].isnan(), w.isnan())
            # as in test_route; the arguments of exp reach 2^128, whose rounding is of results that are 0
            assert ((got[part] - w).abs()[~w.isnan()] <= ((4 + 20 + E) * 2.0 ** -23 * w + 1e-38)[~w.isnan()]).all()
        check_grouping(r.groups, r.ids.flatten(), E)
    # the gradient: 0 where every expert is masked, and at masked experts; the definition's where the weights are numbers
    dw = torch.randn(len(x), k, generator=torch.Generator().manual_seed(k))
    leaf = x.cuda().requires_grad_(True)
    tree_route_topk(leaf, k, renormalize=renormalize).weights.backward(dw.cuda())
    p = torch.zeros(x.shape, dtype=torch.float64).scatter(1, ids, w) if renormalize else torch.softmax(x.double(), 1)
    p = torch.where((x == -math.inf).all(1, keepdim=True), torch.zeros_like(p), p)
    dp = torch.zeros(x.shape, dtype=torch.float64).scatter(1, ids, dw.double())
    want = p * (dp - (p * dp).sum(1, keepdim=True))
    size = p * (dp.abs() + (p * dp.abs()).sum(1, keepdim=True))
    tol = (64 + 2 * E) * 2.0 ** -23 * size + torch.finfo(dtype).eps / 2 * want.abs() + 2.0 ** -25
    fine = ~w.isnan().any(1)
    assert fine.sum() > 10 and ((leaf.grad.cpu().double() - want).abs() <= tol)[fine].all()
    assert (leaf.grad.cpu()[fine][(x == -math.inf)[fine]] == 0).all()


@pytest.mark.parametrize("T", [3, 700])
def test_route_reads_strided_and_broadcast_rows(T):
    from llm_reproducibility_b200.tbik.row_groups import route_topk
    wide = torch.randn(T, 200, device="cuda")
    for x in (wide[:, 17:90], wide[:, ::2], wide[:1, :50].expand(T, 50), wide.t().contiguous().t()[:, :64]):
        r, want = route_topk(x, 5), route_topk(x.contiguous(), 5)
        assert torch.equal(r.ids, want.ids) and torch.equal(r.weights, want.weights) and torch.equal(r.groups.order, want.groups.order)


def test_a_row_is_routed_alike_in_every_batch():
    from llm_reproducibility_b200.tbik.row_groups import route_topk
    x = torch.randn(3000, 96, device="cuda").to(torch.bfloat16)
    full = route_topk(x, 6, renormalize=False)
    for rows in (slice(0, 1), slice(17, 400), slice(1234, 3000)):
        part = route_topk(x[rows], 6, renormalize=False)
        assert torch.equal(part.ids, full.ids[rows]) and torch.equal(part.weights, full.weights[rows])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("T,E,k", [(1, 1, 1), (5, 33, 32), (777, 60, 4), (40, 1024, 32), (513, 128, 8)])
def test_route_gradient(T, E, k, renormalize, dtype):
    from llm_reproducibility_b200.tbik.autograd import tree_route_topk
    g = torch.Generator().manual_seed(E + k)
    x = torch.randn(T, E, generator=g).to(dtype)
    dw = torch.randn(T, k, generator=g)
    leaf = x.cuda().requires_grad_(True)
    r = tree_route_topk(leaf, k, renormalize=renormalize)
    assert not r.ids.requires_grad and not r.groups.order.requires_grad
    r.weights.backward(dw.cuda())
    w, ids = route_ref(x, k, renormalize)
    p = torch.zeros(T, E, dtype=torch.float64)
    p = p.scatter(1, ids, w) if renormalize else torch.softmax(x.double(), 1)
    dp = torch.zeros(T, E, dtype=torch.float64).scatter(1, ids, dw.double())
    want = p * (dp - (p * dp).sum(1, keepdim=True))
    # p's error as above; the bracket's terms are each off by a few units of themselves; then the rounding to the type
    size = p * (dp.abs() + (p * dp.abs()).sum(1, keepdim=True))
    # (a result below fp16's smallest normal number, 2^-14, is off by at most half of its smallest step, 2^-25)
    tol = (64 + 2 * E) * 2.0 ** -23 * size + torch.finfo(dtype).eps / 2 * want.abs() + 2.0 ** -25
    assert leaf.grad.dtype == dtype and ((leaf.grad.cpu().double() - want).abs() <= tol).all()


@pytest.mark.parametrize("renormalize", [True, False])
def test_route_gradient_against_differences(renormalize):
    from llm_reproducibility_b200.tbik.autograd import tree_route_topk
    from llm_reproducibility_b200.tbik.row_groups import route_topk
    x = (torch.arange(24).reshape(2, 12) * 0.37 % 3.0).cuda()      # values well apart: no step changes the choice
    dw = torch.randn(2, 4, generator=torch.Generator().manual_seed(5)).cuda()
    leaf = x.clone().requires_grad_(True)
    tree_route_topk(leaf, 4, renormalize=renormalize).weights.backward(dw)
    h = 2.0 ** -6
    for t in range(2):
        for e in range(12):
            step = torch.zeros_like(x)
            step[t, e] = h
            up, down = (route_topk(x + s, 4, renormalize=renormalize) for s in (step, -step))
            assert torch.equal(up.ids, down.ids)
            diff = ((up.weights.double() - down.weights.double()) * dw).sum() / (2 * h)
            # a softmax's third derivative is at most 1: h^2 / 6 per weight; fp32 weights: 2^-22 / h per weight
            assert abs(diff - leaf.grad[t, e]) <= (h * h / 6 + 2.0 ** -22 / h) * dw[t].abs().sum()


def test_gradient_of_a_masked_row_is_zero():
    from llm_reproducibility_b200.tbik.autograd import tree_route_topk
    for renormalize in (True, False):
        x = torch.full((2, 5), -math.inf)
        x[1, 2] = 1.0
        leaf = x.cuda().requires_grad_(True)
        tree_route_topk(leaf, 2, renormalize=renormalize).weights.backward(torch.ones(2, 2, device="cuda"))
        assert torch.equal(leaf.grad, torch.zeros_like(leaf.grad))


@pytest.mark.parametrize("T", [4, 3000, 20000])
def test_route_on_another_stream_and_in_a_graph(T):
    from llm_reproducibility_b200.tbik.row_groups import route_topk
    x = torch.randn(T, 64, device="cuda")
    want = route_topk(x, 4)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = route_topk(x, 4)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got.groups.order, want.groups.order)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r = route_topk(x, 4)
    for seed in (1, 2):
        x.copy_(torch.randn(T, 64, generator=torch.Generator().manual_seed(seed)))
        graph.replay()
        want = route_topk(x, 4)
        for a, b in zip((r.weights, r.ids, *r.groups), (want.weights, want.ids, *want.groups)):
            assert torch.equal(a, b)


def test_gradient_of_no_tokens():
    from llm_reproducibility_b200.tbik.autograd import tree_route_topk
    x = torch.zeros(0, 8, device="cuda", requires_grad=True)
    r = tree_route_topk(x, 2)
    r.weights.sum().backward()
    assert x.grad.shape == (0, 8) and r.groups.offsets.tolist() == [0] * 9


def test_a_second_derivative_is_refused():
    from llm_reproducibility_b200.tbik.autograd import tree_route_topk
    x = torch.randn(4, 8, device="cuda", requires_grad=True)
    (g,) = torch.autograd.grad(tree_route_topk(x, 2).weights[:, 0].sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()
