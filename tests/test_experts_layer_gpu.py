"""The grouped operators together, as a layer uses them: router, gathered rows, gated up projections, row-split down
projection in the tree, weighted sum of the slots; and adapters beside the tree matmul's shared projection.

The layer is compared with a 64-bit restatement that takes the same roundings (the results of every operator to bf16), so
what is left between the two is each operator's own fp32 work and the roundings that fall to the other side of it."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def weights(E, H, I, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    w = lambda *s: (torch.randn(*s, generator=g, device="cuda") * s[-1] ** -0.5).to(BF16)  # noqa: E731
    return w(E, H), w(E, 2 * I, H), w(E, H, I)


def scores_of(x, gate):
    """[T, E]: the product of one group, which takes any number of experts."""
    from llm_reproducibility_b200.tbik.autograd import tree_grouped_linear
    return tree_grouped_linear(x, gate[None], torch.tensor([0, x.shape[0]], dtype=torch.int32, device=x.device))


def layer(x, gate, up, down, k, tp=1):
    """x [T, H] through k of E experts each; the down projection K-split over tp simulated ranks."""
    from llm_reproducibility_b200.tbik.autograd import tree_grouped_linear, tree_route_topk
    from llm_reproducibility_b200.tbik.grouped_matmul import grouped_matmul_tp_persistent
    from llm_reproducibility_b200.tbik.tree_based_matmul import leaf_for_fp32_nodes
    T, H = x.shape
    r = tree_route_topk(scores_of(x, gate), k)
    rows = x[:, None, :].expand(T, k, H).reshape(T * k, H)[r.groups.order.long()]
    a = tree_grouped_linear(rows, up, r.groups.offsets).float()
    half = a.shape[1] // 2
    act = (torch.nn.functional.silu(a[:, :half]) * a[:, half:]).to(BF16)
    leaf = leaf_for_fp32_nodes(down.shape[2], 8)
    if tp == 1:
        y = tree_grouped_linear(act, down, r.groups.offsets, leaf)
    else:
        ks = down.shape[2] // tp
        parts = [grouped_matmul_tp_persistent(act[:, i * ks:(i + 1) * ks], down[:, :, i * ks:(i + 1) * ks], r.groups.offsets, leaf=leaf,
                                              out_dtype=torch.float32) for i in range(tp)]
        while len(parts) > 1:
            parts = [parts[i] + parts[i + 1] for i in range(0, len(parts), 2)]
        y = parts[0].to(BF16)
    # back to the tokens' order: every token adds its slots in slot order
    mine = y[r.groups.position.long()].view(T, k, H).float()
    return (mine * r.weights[:, :, None]).sum(1).to(BF16)


def restated(x, gate, up, down, ids):
    """The layer in 64 bits on the same parameters, differentiable, with the experts given."""
    d = lambda t: t.double()  # noqa: E731
    w = torch.softmax((x @ gate.t()).gather(1, ids), 1)
    out = torch.zeros_like(x)
    for e in range(gate.shape[0]):
        for j in range(ids.shape[1]):
            rows = torch.nonzero(ids[:, j] == e).flatten()
            a = x[rows] @ d(up[e]).t()
            half = a.shape[1] // 2
            out = out.index_add(0, rows, w[rows, j, None] * ((torch.nn.functional.silu(a[:, :half]) * a[:, half:]) @ d(down[e]).t()))
    return out


@pytest.mark.parametrize("T,E,k,H,I", [(1, 8, 2, 256, 512), (37, 8, 3, 512, 512), (700, 16, 4, 256, 1024)])
def test_layer_and_its_gradients(T, E, k, H, I):
    from llm_reproducibility_b200.tbik.row_groups import route_topk
    gate, up, down = weights(E, H, I, 3)
    x = torch.randn(T, H, generator=torch.Generator(device="cuda").manual_seed(T), device="cuda").to(BF16)
    dy = torch.randn(T, H, generator=torch.Generator(device="cuda").manual_seed(T + 1), device="cuda").to(BF16)
    params = [t.clone().requires_grad_(True) for t in (x, gate, up, down)]
    out = layer(*params, k)
    grads = torch.autograd.grad(out, params, dy)
    exact = [t.double().requires_grad_(True) for t in (x, gate, up, down)]
    with torch.no_grad():
        ids = route_topk(scores_of(x, gate), k).ids.long()  # (which experts: tests/test_row_groups_gpu.py)
    want = restated(*exact, ids)
    wants = torch.autograd.grad(want, exact, dy.double())
    # A value of the layer has passed at most six roundings to bf16 (scores, up, activation, down, sum, result), one of its
    # gradients as many again, each off by at most 2^-8 of the value: in the 2-norm 12 x 2^-8 of the result were all of them
    # at their worst and of one sign (the fp32 work is below 2^-14).  The gate's gradient is a difference, p (dp - <p, dp>),
    # whose terms with random scores and gradients are no larger than itself in the 2-norm over the tokens.
    for got, ref in zip([out] + list(grads), [want] + list(wants)):
        assert (got.double() - ref).norm() <= 12 * 2.0 ** -8 * ref.norm()


def test_layer_is_batch_and_tensor_parallel_invariant():
    gate, up, down = weights(16, 256, 1024, 5)
    x = torch.randn(600, 256, generator=torch.Generator(device="cuda").manual_seed(9), device="cuda").to(BF16)
    with torch.no_grad():
        full = layer(x, gate, up, down, 4)
        for tp in (2, 4, 8):
            assert torch.equal(layer(x, gate, up, down, 4, tp), full), tp
        for rows in (slice(0, 1), slice(3, 20), slice(100, 600)):
            assert torch.equal(layer(x[rows], gate, up, down, 4), full[rows])


def test_adapters_beside_the_shared_projection():
    """The row-split layer with adapters: shards of x and A, the shared projection's and the adapters' sums joined in the
    rank-pair tree: the unsharded bits at every degree, and the same row bits in every batch."""
    from llm_reproducibility_b200.tbik.adapters import leaf_for_adapters, lora_add, lora_expand_add, lora_shrink
    from llm_reproducibility_b200.tbik.row_groups import group_rows
    from llm_reproducibility_b200.tbik.tree_based_matmul import leaf_for, matmul_tp_persistent
    T, K, N, L, R = 90, 4096, 512, 5, 16
    g = torch.Generator(device="cuda").manual_seed(1)
    x, W = torch.randn(T, K, generator=g, device="cuda").to(BF16), (torch.randn(N, K, generator=g, device="cuda") / 64).to(BF16)
    A, B = (torch.randn(L, R, K, generator=g, device="cuda") / 64).to(BF16), torch.randn(L, N, R, generator=g, device="cuda").to(BF16)
    ids = torch.randint(-1, L, (T,), generator=g, device="cuda").to(torch.int32)
    scales = torch.rand(L, generator=g, device="cuda")
    leaf = leaf_for(K)

    def tree(parts):
        while len(parts) > 1:
            parts = [parts[i] + parts[i + 1] for i in range(0, len(parts), 2)]
        return parts[0]

    def forward(rows, tp):
        groups, ks = group_rows(ids[rows], L), K // tp
        cut = [slice(r * ks, (r + 1) * ks) for r in range(tp)]
        y = tree([matmul_tp_persistent(x[rows][:, c], W[:, c].t(), leaf=leaf) for c in cut])
        if tp == 1:
            return lora_add(y, x[rows], A, B, groups, scales)
        h = tree([lora_shrink(x[rows][:, c], A[:, :, c], groups, leaf=leaf_for_adapters(K)) for c in cut])
        return lora_expand_add(y, h, B, groups, scales)

    full = forward(slice(0, T), 1)
    for tp in (2, 4, 8):
        assert torch.equal(forward(slice(0, T), tp), full)
    for rows in (slice(0, 1), slice(7, 30)):
        for tp in (1, 4):
            assert torch.equal(forward(rows, tp), full[rows])
    plain = matmul_tp_persistent(x, W.t(), leaf=leaf)
    assert torch.equal(full[ids < 0], plain[ids < 0]) and not torch.equal(full[ids >= 0], plain[ids >= 0])


@pytest.mark.parametrize("what", ["grouped", "lora_add", "lora_expand_add"])
def test_a_saved_tensor_that_is_overwritten_is_noticed(what):
    """What autograd saved and a kernel then overwrote must not pass for the gradient."""
    from llm_reproducibility_b200.tbik.adapters import lora_add, lora_expand_add
    from llm_reproducibility_b200.tbik.grouped_matmul import grouped_matmul_tp_persistent
    from llm_reproducibility_b200.tbik.row_groups import group_rows
    ones = lambda *s: torch.ones(*s, dtype=torch.bfloat16, device="cuda")  # noqa: E731
    groups, scales = group_rows(torch.zeros(4, dtype=torch.int32, device="cuda"), 1), torch.ones(1, device="cuda")
    leaf, y = ones(4, 16).requires_grad_(True), ones(4, 16)
    z = (leaf * y).sum()  # y is saved for leaf's gradient
    before = y._version
    if what == "grouped":
        got = grouped_matmul_tp_persistent(ones(4, 64), ones(1, 16, 64), groups.offsets, out=y)
    elif what == "lora_add":
        got = lora_add(y, ones(4, 64), ones(1, 8, 64), ones(1, 16, 8), groups, scales, out=y)
    else:
        got = lora_expand_add(y, torch.ones(4, 8, device="cuda"), ones(1, 16, 8), groups, scales, out=y)
    assert got is y and y._version > before
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        z.backward()
    with torch.inference_mode():  # tensors without a version
        y = ones(4, 16)
        assert lora_expand_add(y, torch.ones(4, 8, device="cuda"), ones(1, 16, 8), groups, scales, out=y) is y
    assert lora_expand_add(y, torch.ones(4, 8, device="cuda"), ones(1, 16, 8), groups, scales, out=y) is y and (y == 17).all()
