"""Products grouped by expert: forward, input gradient and weight gradient against 64-bit restatements, over ragged and
empty groups, odd sizes, layouts, types and the sizes at which the kernels change their form.

Two kinds of operands.  Small integers: every product and sum is exact in fp32 in any order, so the result has to be the
exact value rounded once, bit for bit.  Normal deviates: |error| <= eps/2 |value| for the rounding plus, for n terms added
in fp32 by an adder that may truncate, n 2^-23 times the sum of the terms' magnitudes."""
import pytest
import torch

pytestmark = pytest.mark.gpu

HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def offsets_of(sizes, lead=0):
    return torch.tensor([lead] + list(sizes)).cumsum(0).to(torch.int32)


def ragged(M, G, seed):
    """G sizes that add up to M, uneven, some empty."""
    g = torch.Generator().manual_seed(seed)
    p = torch.rand(G, generator=g) ** 3
    ids = torch.multinomial(p, M, replacement=True, generator=g) if M else torch.zeros(0, dtype=torch.long)
    return torch.bincount(ids, minlength=G).tolist()


def make(shape, dtype, kind, seed, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    if kind == "int":
        return torch.randint(-3, 4, shape, generator=g, device="cuda").to(dtype)
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def forward_ref(A, W, offsets):
    """(value, sum of magnitudes) in fp64; rows of no group are zero."""
    C = torch.zeros(A.shape[0], W.shape[1], dtype=torch.float64, device=A.device)
    S = torch.zeros_like(C)
    at = offsets.tolist()
    for g, (lo, hi) in enumerate(zip(at, at[1:])):
        a, w = A[lo:hi].double(), W[g].double()
        C[lo:hi], S[lo:hi] = a @ w.t(), a.abs() @ w.abs().t()
    return C, S


def wgrad_ref(D, A, offsets):
    at = offsets.tolist()
    out = [(D[lo:hi].double().t() @ A[lo:hi].double(), D[lo:hi].double().abs().t() @ A[lo:hi].double().abs(), hi - lo)
           for lo, hi in zip(at, at[1:])]
    return torch.stack([o[0] for o in out]), torch.stack([o[1] * o[2] for o in out])


def check(got, value, size, kind, n_terms=1):
    if kind == "int":
        assert torch.equal(got, value.to(got.dtype)), (got.double() - value).abs().max()
    else:
        tol = HALF[got.dtype] * value.abs() + n_terms * 2.0 ** -23 * size + 2.0 ** -25
        bad = (got.double() - value).abs() > tol
        assert not bad.any(), (int(bad.sum()), ((got.double() - value).abs() - tol).max())


# (rows, groups, K, N): one row; small tiles; odd K and N; sizes around tile borders; enough rows for every row tile
SHAPES = [(1, 1, 64, 64), (1, 128, 64, 40), (8, 16, 256, 128), (5, 3, 13, 7), (37, 4, 72, 100), (130, 2, 520, 257), (128, 1, 64, 128),
          (257, 5, 192, 192), (1000, 7, 104, 1000), (700, 64, 512, 96), (2500, 3, 320, 384), (4099, 6, 136, 512), (6000, 2, 256, 768)]


@pytest.mark.parametrize("kind", ["int", "normal"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M,G,K,N", SHAPES)
def test_forward(M, G, K, N, dtype, kind):
    from llm_reproducibility_b200.tbik.grouped_matmul import grouped_matmul_tp_persistent
    A, W = make((M, K), dtype, kind, 1), make((G, N, K), dtype, kind, 2, 0.1)
    off = offsets_of(ragged(M, G, M + K)).cuda()
    value, size = forward_ref(A, W, off)
    check(grouped_matmul_tp_persistent(A, W, off), value, size, kind, K)
    check(grouped_matmul_tp_persistent(A, W, off, out_dtype=torch.float32), value, size, kind, K)


@pytest.mark.parametrize("kind", ["int", "normal"])
@pytest.mark.parametrize("M,G,K,N", SHAPES)
def test_forward_with_a_transposed_weight(M, G, K, N, kind):
    """W given as the [G, N, K] view of [G, K, N] memory."""
    from llm_reproducibility_b200.tbik.grouped_matmul import grouped_matmul_tp_persistent
    A, W = make((M, K), torch.bfloat16, kind, 3), make((G, K, N), torch.bfloat16, kind, 4, 0.1).transpose(1, 2)
    off = offsets_of(ragged(M, G, M + N)).cuda()
    value, size = forward_ref(A, W, off)
    check(grouped_matmul_tp_persistent(A, W, off), value, size, kind, K)


@pytest.mark.parametrize("kind", ["int", "normal"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M,G,K,N", SHAPES)
def test_weight_gradient(M, G, K, N, dtype, kind):
    from llm_reproducibility_b200.tbik.grouped_matmul import grouped_weight_gradient
    D, A = make((M, N), dtype, kind, 5, 0.3), make((M, K), dtype, kind, 6)
    off = offsets_of(ragged(M, G, M + N + K)).cuda()
    value, size = wgrad_ref(D, A, off)
    check(grouped_weight_gradient(D, A, off), value, size, kind)
    check(grouped_weight_gradient(D, A, off, out_dtype=torch.float32), value, size, kind)


@pytest.mark.parametrize("sizes", [[0, 0, 0], [0, 5, 0], [1, 1, 1], [128, 128, 128], [127, 129, 1], [64, 0, 300], [15, 17, 16], [256, 255, 257]])
@pytest.mark.parametrize("lead,tail", [(0, 0), (3, 70)])
def test_group_borders_and_rows_of_no_group(sizes, lead, tail):
    """Rows before the first and behind the last group: zero in a new result, untouched in `out`, absent from dW --
    also when they hold NaN."""
    from llm_reproducibility_b200.tbik.grouped_matmul import grouped_matmul_tp_persistent, grouped_weight_gradient
    K, N, M = 96, 160, lead + sum(sizes) + tail
    if M == 0:
        M = 1
    A, W, D = make((M, K), torch.bfloat16, "int", 7), make((3, N, K), torch.bfloat16, "int", 8), make((M, N), torch.bfloat16, "int", 9)
    off = offsets_of(sizes, lead).cuda()
    first, last = lead, lead + sum(sizes)
    value, _ = forward_ref(A, W, off)
    dvalue, _ = wgrad_ref(D, A, off)
    for t in (A, D):
        t[:first], t[last:] = float("nan"), float("nan")
    got = grouped_matmul_tp_persistent(A, W, off)
    assert torch.equal(got, value.to(torch.bfloat16))
    out = torch.full((M, N), 7.0, dtype=torch.bfloat16, device="cuda")
    grouped_matmul_tp_persistent(A, W, off, out=out)
    assert torch.equal(out[first:last], got[first:last]) and (out[:first] == 7).all() and (out[last:] == 7).all()
    assert torch.equal(grouped_weight_gradient(D, A, off), dvalue.to(torch.bfloat16))


def test_a_group_with_nan_leaves_the_others_alone():
    from llm_reproducibility_b200.tbik.grouped_matmul import grouped_matmul_tp_persistent, grouped_weight_gradient
    sizes, K, N = [70, 33, 90, 0, 5], 128, 128
    off, M = offsets_of(sizes).cuda(), sum(sizes)
    A, W, D = make((M, K), torch.bfloat16, "int", 1), make((5, N, K), torch.bfloat16, "int", 2), make((M, N), torch.bfloat16, "int", 3)
    fwd, grad = forward_ref(A, W, off)[0].to(torch.bfloat16), wgrad_ref(D, A, off)[0].to(torch.bfloat16)
    for bad in (float("nan"), float("inf")):
        A2, W2, D2 = A.clone(), W.clone(), D.clone()
        A2[70:103], D2[70:103], W2[1] = bad, bad, bad
        C = grouped_matmul_tp_persistent(A2, W2, off)
        dW = grouped_weight_gradient(D2, A2, off)
        keep = [i for i in range(M) if not 70 <= i < 103]
        assert torch.equal(C[keep], fwd[keep]) and not C[70:103].isfinite().any()
        assert torch.equal(dW[[0, 2, 3, 4]], grad[[0, 2, 3, 4]])


@pytest.mark.parametrize("w_n_contiguous", [False, True])
@pytest.mark.parametrize("K,leaf", [(512, 64), (768, 192), (4096, 512), (1536, 256), (64, 64), (2048, 128), (16384, 64)])
def test_tree_over_k(K, leaf, w_n_contiguous):
    """The leaves' sums are joined in the framework's tree: same value, and shards of K add up to the unsharded bits."""
    from llm_reproducibility_b200.tbik.grouped_matmul import grouped_matmul_tp_persistent
    from llm_reproducibility_b200.tbik.tree_based_matmul import tree_shape
    M, G, N = 300, 4, 200
    A, W = make((M, K), torch.bfloat16, "normal", 11), make((G, N, K), torch.bfloat16, "normal", 12, 0.1)
    if w_n_contiguous:
        W = W.transpose(1, 2).contiguous().transpose(1, 2)
    off = offsets_of(ragged(M, G, 5)).cuda()
    value, size = forward_ref(A, W, off)
    full = grouped_matmul_tp_persistent(A, W, off, leaf=leaf)
    check(full, value, size, "normal", K)
    root = grouped_matmul_tp_persistent(A, W, off, leaf=leaf, out_dtype=torch.float32)
    assert torch.equal(root.to(torch.bfloat16), full)
    T, F, L = tree_shape(K, leaf)
    for tp in (2, 4, 8):
        if (1 << (L - 1)) % tp:
            continue
        ks = K // tp
        parts = [grouped_matmul_tp_persistent(A[:, r * ks:(r + 1) * ks], W[:, :, r * ks:(r + 1) * ks], off, leaf=leaf,
                                              out_dtype=torch.float32) for r in range(tp)]
        while len(parts) > 1:
            parts = [parts[i] + parts[i + 1] for i in range(0, len(parts), 2)]
        assert torch.equal(parts[0], root), tp


def test_a_row_has_the_same_bits_in_every_batch_and_grid():
    from llm_reproducibility_b200.tbik.grouped_matmul import grouped_matmul_tp_persistent
    G, K, N = 3, 512, 320
    A, W = make((3000, K), torch.bfloat16, "normal", 1), make((G, N, K), torch.bfloat16, "normal", 2, 0.1)
    off = torch.tensor([0, 1500, 1501, 3000], dtype=torch.int32, device="cuda")
    full = grouped_matmul_tp_persistent(A, W, off)
    for rows, o in ((slice(100, 101), [0, 1, 1, 1]), (slice(1400, 1600), [0, 100, 101, 200]), (slice(1500, 1516), [0, 0, 1, 16])):
        part = grouped_matmul_tp_persistent(A[rows], W, torch.tensor(o, dtype=torch.int32, device="cuda"))
        assert torch.equal(part, full[rows])
    for ctas in (1, 2, 7, 64):
        assert torch.equal(grouped_matmul_tp_persistent(A, W, off, max_ctas=ctas), full)


def test_weight_gradient_depends_on_the_groups_own_rows_and_not_on_the_grid():
    from llm_reproducibility_b200.tbik.grouped_matmul import grouped_weight_gradient
    D, A = make((900, 264), torch.bfloat16, "normal", 1), make((900, 136), torch.bfloat16, "normal", 2)
    off = torch.tensor([0, 317, 317, 900], dtype=torch.int32, device="cuda")
    full = grouped_weight_gradient(D, A, off)
    alone = grouped_weight_gradient(D[317:], A[317:], torch.tensor([0, 583], dtype=torch.int32, device="cuda"))
    assert torch.equal(full[2], alone[0]) and (full[1] == 0).all()
    for ctas in (1, 2, 9):
        assert torch.equal(grouped_weight_gradient(D, A, off, max_ctas=ctas), full)


@pytest.mark.parametrize("N,K,sizes,ctas", [(38400, 64, [103, 97], 1), (8192, 64, [3, 0, 17, 5, 1, 16, 2, 9], 1), (520, 64, [30] * 600, 3)])
def test_more_tiles_than_are_worked_out_ahead(N, K, sizes, ctas):
    """Hundreds of tiles for one CTA, or one pair: the ones beyond the first 256 are found as they come."""
    from llm_reproducibility_b200.tbik.grouped_matmul import grouped_matmul_tp_persistent, grouped_weight_gradient
    off = offsets_of(sizes).cuda()
    A, W = make((sum(sizes), K), torch.bfloat16, "int", 1), make((len(sizes), N, K), torch.bfloat16, "int", 2)
    got = grouped_matmul_tp_persistent(A, W, off, max_ctas=ctas)
    assert torch.equal(got, forward_ref(A, W, off)[0].to(torch.bfloat16))
    for n, k in ((2048, 2048), (100, 2304)):  # tiles of a pair, of one CTA
        D, A = make((sum(sizes[:8]), n), torch.bfloat16, "int", 3), make((sum(sizes[:8]), k), torch.bfloat16, "int", 4)
        some = torch.cat([off[:9], off[8:9].expand(24)]) if len(sizes) > 8 else off
        some = some.clamp(max=D.shape[0]).contiguous()
        want = wgrad_ref(D, A, some)[0].to(torch.bfloat16)
        assert torch.equal(grouped_weight_gradient(D, A, some, max_ctas=ctas), want)


@pytest.mark.parametrize("N,K", [(264, 136), (100, 520)])
def test_weight_gradient_of_a_group_beside_infinities_and_nan(N, K):
    """The rows behind a group's last step of 16 come along with it and belong to someone else."""
    from llm_reproducibility_b200.tbik.grouped_matmul import grouped_weight_gradient
    sizes = [1, 1, 15, 3, 16, 2, 17, 1, 63, 9, 64, 5, 65, 4, 130, 7]
    off = offsets_of(sizes).cuda()
    D, A = make((sum(sizes), N), torch.bfloat16, "int", 1), make((sum(sizes), K), torch.bfloat16, "int", 2)
    want = wgrad_ref(D, A, off)[0].to(torch.bfloat16)
    at = off.tolist()
    for g in range(1, len(sizes), 2):
        D[at[g]:at[g + 1]] = float("nan")
        A[at[g]:at[g + 1]] = float("inf")
    for ctas in (0, 2):
        got = grouped_weight_gradient(D, A, off, max_ctas=ctas)
        assert torch.equal(got[::2], want[::2]) and got[1::2].isnan().all()


def test_strided_and_unaligned_operands():
    from llm_reproducibility_b200.tbik.grouped_matmul import grouped_matmul_tp_persistent, grouped_weight_gradient
    M, G, K, N = 200, 3, 64, 48
    off = offsets_of([50, 100, 50]).cuda()
    big = make((M + 1, 3 * K + 5), torch.bfloat16, "int", 1)
    wbig = make((G, N + 3, 2 * K + 1), torch.bfloat16, "int", 2)
    dbig = make((M, 2 * N + 3), torch.bfloat16, "int", 3)
    for A in (big[:M, :K], big[1:, 3:3 + K], big[:M, 0:2 * K:2], big.t()[:K, :].t()[:M], big[:1, :K].expand(M, K)):
        for W in (wbig[:, :N, :K], wbig[:, 1:N + 1, 1:K + 1], wbig[:1, :N, :K].expand(G, N, K), wbig[:, ::1, ::2][:, :N, :K]):
            want = forward_ref(A, W, off)[0].to(torch.bfloat16)
            assert torch.equal(grouped_matmul_tp_persistent(A, W, off), want)
        for D in (dbig[:, :N], dbig[:, 1:2 * N:2], dbig[:1, :N].expand(M, N)):
            assert torch.equal(grouped_weight_gradient(D, A, off), wgrad_ref(D, A, off)[0].to(torch.bfloat16))


@pytest.mark.parametrize("M,G,K,N", [(200, 3, 64, 48), (9, 4, 520, 264), (3000, 2, 320, 384), (40, 5, 13, 7)])
def test_weights_whose_groups_lie_row_by_row_in_turn(M, G, K, N):
    """[N, G, K] and [K, G, N] memory seen as [G, N, K], windows that overlap, forward and backward: the copied weight's bits."""
    from llm_reproducibility_b200.tbik.autograd import tree_grouped_linear
    from llm_reproducibility_b200.tbik.grouped_matmul import grouped_matmul_tp_persistent
    off = offsets_of(ragged(M, G, M)).cuda()
    A, D = make((M, K), torch.bfloat16, "normal", 1), make((M, N), torch.bfloat16, "normal", 2)
    nested = make((N, G, K), torch.bfloat16, "normal", 3).permute(1, 0, 2)
    other = make((K, G, N), torch.bfloat16, "normal", 4).permute(1, 2, 0)
    step = (K + 7) // 8 * 8
    window = make((G * (step + 8) + N * step,), torch.bfloat16, "normal", 5).as_strided((G, N, K), (step + 8, step, 1))
    for W in (nested, other, window):
        want = grouped_matmul_tp_persistent(A, W.contiguous(), off)
        check(want, *forward_ref(A, W, off), "normal", K)
        assert torch.equal(grouped_matmul_tp_persistent(A, W, off), want)
        x, w, w2 = A.clone().requires_grad_(True), W.detach().requires_grad_(True), W.contiguous().requires_grad_(True)
        got = torch.autograd.grad(tree_grouped_linear(x, w, off), (x, w), D)
        for g, v in zip(got, torch.autograd.grad(tree_grouped_linear(x, w2, off), (x, w2), D)):
            assert torch.equal(g, v)
    if K % 64 == 0:
        leaf = K // (K // 64)
        assert torch.equal(grouped_matmul_tp_persistent(A, nested, off, leaf=leaf), grouped_matmul_tp_persistent(A, nested.contiguous(), off, leaf=leaf))


@pytest.mark.parametrize("M,N", [(5, 0), (0, 7), (0, 0)])
def test_gradients_of_no_columns_and_of_no_rows(M, N):
    from llm_reproducibility_b200.tbik.autograd import tree_grouped_linear
    x, w = (make(s, torch.bfloat16, "int", 1).requires_grad_(True) for s in ((M, 64), (2, N, 64)))
    y = tree_grouped_linear(x, w, offsets_of([M // 2, M - M // 2]).cuda())
    dx, dw = torch.autograd.grad(y, (x, w), torch.ones(M, N, dtype=torch.bfloat16, device="cuda"))
    assert y.shape == (M, N) and torch.equal(dx, torch.zeros_like(x)) and torch.equal(dw, torch.zeros_like(w))


def test_out_with_a_wide_stride_and_neighbours_untouched():
    from llm_reproducibility_b200.tbik.grouped_matmul import grouped_matmul_tp_persistent
    for M, N, wide in ((300, 128, 160), (300, 100, 101), (77, 7, 9), (1, 40, 64)):
        A, W = make((M, 64), torch.bfloat16, "int", 1), make((2, N, 64), torch.bfloat16, "int", 2)
        off = offsets_of([M // 3, M - M // 3]).cuda()
        buf = torch.full((M + 2, wide), 5.0, dtype=torch.bfloat16, device="cuda")
        grouped_matmul_tp_persistent(A, W, off, out=buf[1:M + 1, 1:N + 1])
        assert torch.equal(buf[1:M + 1, 1:N + 1], forward_ref(A, W, off)[0].to(torch.bfloat16))
        buf[1:M + 1, 1:N + 1] = 5.0
        assert (buf == 5.0).all()


def test_bad_tables_touch_nothing_outside():
    """A table is read by the kernels alone: whatever it holds, only rows of C are written."""
    from llm_reproducibility_b200.tbik.grouped_matmul import grouped_matmul_tp_persistent, grouped_weight_gradient
    M, K, N = 100, 64, 64
    A, W, D = make((M, K), torch.bfloat16, "int", 1), make((3, N, K), torch.bfloat16, "int", 2), make((M, N), torch.bfloat16, "int", 3)
    for table in ([0, 2 ** 31 - 1, 2 ** 31 - 1, 2 ** 31 - 1], [-5, -1, 50, 400], [0, 70, 20, 100], [2 ** 31 - 1, 0, 0, 0], [-2 ** 31] * 4):
        off = torch.tensor(table, dtype=torch.int64).to(torch.int32).cuda()
        buf = torch.full((M + 2, N), 5.0, dtype=torch.bfloat16, device="cuda")
        grouped_matmul_tp_persistent(A, W, off, out=buf[1:M + 1])
        grouped_weight_gradient(D, A, off)
        assert (buf[0] == 5).all() and (buf[-1] == 5).all()
    assert grouped_matmul_tp_persistent(A[:0], W, torch.zeros(4, dtype=torch.int32, device="cuda")).shape == (0, N)
    assert (grouped_weight_gradient(D[:0], A[:0], torch.zeros(4, dtype=torch.int32, device="cuda")) == 0).all()


@pytest.mark.parametrize("M,G,K,N", [(37, 4, 72, 100), (300, 3, 128, 256), (9, 2, 13, 7)])
def test_gradients_through_autograd(M, G, K, N):
    """Against the formulas, and -- the product being bilinear and the operands small integers -- against exact differences."""
    from llm_reproducibility_b200.tbik.autograd import tree_grouped_linear
    x, w = make((M, K), torch.bfloat16, "int", 1).requires_grad_(True), make((G, N, K), torch.bfloat16, "int", 2).requires_grad_(True)
    dy = make((M, N), torch.bfloat16, "int", 3)
    off = offsets_of(ragged(M - 4, G, 9), 2).cuda()  # two rows of no group in front, two behind
    y = tree_grouped_linear(x, w, off)
    y.backward(dy)
    dx = torch.zeros(M, K, dtype=torch.float64, device="cuda")
    at = off.tolist()
    for g, (lo, hi) in enumerate(zip(at, at[1:])):
        dx[lo:hi] = dy[lo:hi].double() @ w[g].detach().double()
    assert torch.equal(x.grad, dx.to(torch.bfloat16))
    assert torch.equal(w.grad, wgrad_ref(dy, x.detach(), off)[0].to(torch.bfloat16))
    from llm_reproducibility_b200.tbik.grouped_matmul import grouped_matmul_tp_persistent
    loss = lambda a, b: float((grouped_matmul_tp_persistent(a, b, off, out_dtype=torch.float32).double() * dy.double()).sum())  # noqa: E731
    xd, wd = x.detach(), w.detach()
    base = loss(xd, wd)
    for i, k in ((0, 0), (M // 2, K - 1), (M - 3, 1), (M - 1, 0)):
        x2 = xd.clone()
        x2[i, k] += 1
        assert loss(x2, wd) - base == float(dx[i, k])
    exact = wgrad_ref(dy, xd, off)[0]
    for g, n, k in ((0, 0, 0), (G - 1, N - 1, K - 1), (G // 2, N // 2, 0)):
        w2 = wd.clone()
        w2[g, n, k] += 1
        assert loss(xd, w2) - base == float(exact[g, n, k])


def test_gradients_only_where_asked_and_of_shared_leaves():
    from llm_reproducibility_b200.tbik.autograd import tree_grouped_linear
    off = offsets_of([20, 30]).cuda()
    x, w = make((50, 64), torch.bfloat16, "int", 1), make((2, 64, 64), torch.bfloat16, "int", 2)
    dy = make((50, 64), torch.bfloat16, "int", 3)
    for gx, gw in ((True, False), (False, True)):
        a, b = x.clone().requires_grad_(gx), w.clone().requires_grad_(gw)
        tree_grouped_linear(a, b, off).backward(dy)
        assert (a.grad is not None) == gx and (b.grad is not None) == gw
    # one weight for both groups: its gradient is the sum over the broadcast
    one = w[:1].clone().requires_grad_(True)
    tree_grouped_linear(x, one.expand(2, 64, 64), off).backward(dy)
    want = wgrad_ref(dy, x, off)[0].to(torch.bfloat16)
    assert torch.equal(one.grad[0], want[0] + want[1])
    # a loss that is a sum: its gradient arrives as an expanded scalar
    a = x.clone().requires_grad_(True)
    tree_grouped_linear(a, w, off).float().sum().backward()
    assert a.grad.isfinite().all()


def test_two_streams_and_a_graph():
    from llm_reproducibility_b200.tbik.grouped_matmul import grouped_matmul_tp_persistent, grouped_weight_gradient
    off = offsets_of([100, 0, 200]).cuda()
    A, W, D = make((300, 256), torch.bfloat16, "int", 1), make((3, 128, 256), torch.bfloat16, "int", 2), make((300, 128), torch.bfloat16, "int", 3)
    want, dwant = grouped_matmul_tp_persistent(A, W, off), grouped_weight_gradient(D, A, off)
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            outs.append([(grouped_matmul_tp_persistent(A, W, off), grouped_weight_gradient(D, A, off)) for _ in range(4)])
    torch.cuda.synchronize()
    assert all(torch.equal(c, want) and torch.equal(d, dwant) for o in outs for c, d in o)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c, d = grouped_matmul_tp_persistent(A, W, off), grouped_weight_gradient(D, A, off)
    # the captured call follows a new table: the kernels read it, not the host
    off.copy_(torch.tensor([0, 7, 250, 290], dtype=torch.int32))
    graph.replay()
    assert torch.equal(c, forward_ref(A, W, off)[0].to(torch.bfloat16)) and torch.equal(d, wgrad_ref(D, A, off)[0].to(torch.bfloat16))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("sizes,K,N,leaf", [([1, 7, 16, 17, 33], 512, 384, 512), ([64, 0, 65, 128, 129], 1024, 256, 128),
                                            ([300, 1, 1000], 768, 640, 96 * 8), ([700, 500], 2048, 512, 256), ([5, 6], 4096, 1024, 512),
                                            ([40, 50], 2048, 128, 64)])
def test_a_groups_rows_have_the_dense_products_bits(sizes, K, N, leaf, dtype):
    from llm_reproducibility_b200.tbik.grouped_matmul import grouped_matmul_tp_persistent
    from llm_reproducibility_b200.tbik.tree_based_matmul import matmul_tp_persistent
    M, G = sum(sizes), len(sizes)
    A, W = make((M, K), dtype, "normal", 21), make((G, N, K), dtype, "normal", 22, 0.1)
    off = offsets_of(sizes).cuda()
    got = grouped_matmul_tp_persistent(A, W, off, leaf=leaf)
    if leaf == K:
        assert torch.equal(got, grouped_matmul_tp_persistent(A, W, off))  # K is one leaf by default
    for g, (lo, hi) in enumerate(zip(off.tolist(), off.tolist()[1:])):
        if hi > lo:
            assert torch.equal(got[lo:hi], matmul_tp_persistent(A[lo:hi], W[g].t(), node_dtype=torch.float32, leaf=leaf)), g


def test_device_status_stays_clean():
    from llm_reproducibility_b200.tbik.tree_based_matmul import gemm_device_status
    torch.cuda.synchronize()
    assert gemm_device_status()[0] == 0


def test_first_cuda_call_of_a_host_thread():
    """A backward pass runs in a thread of its own, whose first CUDA call may be this one: nothing before it may have
    bound a context there (the allocator serves the result from its cache)."""
    import threading
    from llm_reproducibility_b200.tbik.grouped_matmul import grouped_matmul_tp_persistent, grouped_weight_gradient
    off = offsets_of([20, 30]).cuda()
    A, W, D = make((50, 64), torch.bfloat16, "int", 1), make((2, 72, 64), torch.bfloat16, "int", 2), make((50, 72), torch.bfloat16, "int", 3)
    want, dwant = grouped_matmul_tp_persistent(A, W, off), grouped_weight_gradient(D, A, off)
    spare = [torch.empty_like(want), torch.empty_like(dwant)]
    del spare
    torch.cuda.synchronize()
    for call, expected in ((lambda: grouped_matmul_tp_persistent(A, W, off), want), (lambda: grouped_weight_gradient(D, A, off), dwant)):
        got = []

        def work():
            try:
                got.append(call())
            except Exception as e:  # noqa: BLE001
                got.append(e)

        t = threading.Thread(target=work)
        t.start()
        t.join()
        torch.cuda.synchronize()
        assert torch.is_tensor(got[0]) and torch.equal(got[0], expected), got[0]


def test_results_beyond_32_bit_offsets():
    """More than 2^31 elements in C and in dW."""
    from llm_reproducibility_b200.tbik.grouped_matmul import grouped_matmul_tp_persistent, grouped_weight_gradient
    M, N, K = 270000, 8192, 16
    A, W = make((M, K), torch.bfloat16, "int", 1), make((3, N, K), torch.bfloat16, "int", 2)
    off = torch.tensor([0, 100000, 262200, M - 5], dtype=torch.int32, device="cuda")
    C = grouped_matmul_tp_persistent(A, W, off)
    for g, rows in ((0, slice(0, 40)), (1, slice(262144, 262200)), (2, slice(M - 60, M - 5))):
        assert torch.equal(C[rows], (A[rows].double() @ W[g].double().t()).to(torch.bfloat16))
    assert (C[M - 5:] == 0).all()
    del C
    D, X = make((64, 33000), torch.bfloat16, "int", 3), make((64, 33000), torch.bfloat16, "int", 4)
    dW = grouped_weight_gradient(D, X, torch.tensor([0, 10, 64], dtype=torch.int32, device="cuda"))
    assert dW.numel() > 1 << 31
    for g, (lo, hi) in enumerate(((0, 10), (10, 64))):
        for n in (0, 32999):
            assert torch.equal(dW[g, n], (D[lo:hi, n].double() @ X[lo:hi].double()).to(torch.bfloat16))


def test_forward_and_gradients_captured_in_a_graph():
    from llm_reproducibility_b200.tbik.autograd import tree_grouped_linear
    off = offsets_of([70, 0, 130]).cuda()
    x, w = make((200, 128), torch.bfloat16, "int", 1).requires_grad_(True), make((3, 256, 128), torch.bfloat16, "int", 2).requires_grad_(True)
    dy = make((200, 256), torch.bfloat16, "int", 3)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(tree_grouped_linear(x, w, off), (x, w), dy)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = tree_grouped_linear(x, w, off)
        dx, dw = torch.autograd.grad(y, (x, w), dy)
    with torch.no_grad():
        x.copy_(make((200, 128), torch.bfloat16, "int", 7))
        off.copy_(torch.tensor([0, 33, 150, 199], dtype=torch.int32))
    graph.replay()
    assert torch.equal(y, forward_ref(x.detach(), w.detach(), off)[0].to(torch.bfloat16))
    assert torch.equal(dw, wgrad_ref(dy, x.detach(), off)[0].to(torch.bfloat16))
    at = off.tolist()
    for g, (lo, hi) in enumerate(zip(at, at[1:])):
        assert torch.equal(dx[lo:hi], (dy[lo:hi].double() @ w[g].detach().double()).to(torch.bfloat16))
    assert (dx[199:] == 0).all()


def test_no_rows_at_all_and_second_derivatives():
    from llm_reproducibility_b200.tbik.autograd import tree_grouped_linear
    w = make((2, 16, 8), torch.bfloat16, "int", 1).requires_grad_(True)
    x = torch.zeros(0, 8, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    tree_grouped_linear(x, w, torch.zeros(3, dtype=torch.int32, device="cuda")).sum().backward()
    assert x.grad.shape == (0, 8) and (w.grad == 0).all()
    x = make((4, 8), torch.bfloat16, "int", 2).requires_grad_(True)
    (g,) = torch.autograd.grad(tree_grouped_linear(x, w, offsets_of([2, 2]).cuda()).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_refusals_on_the_device():
    from llm_reproducibility_b200.tbik.grouped_matmul import grouped_matmul_tp_persistent as f
    A, W, off = make((8, 64), torch.bfloat16, "int", 1), make((2, 64, 64), torch.bfloat16, "int", 2), offsets_of([4, 4]).cuda()
    with pytest.raises(RuntimeError, match="CUDA"):
        f(A, W, off.cpu())
    for out in (torch.empty(8, 63, dtype=torch.bfloat16, device="cuda"), torch.empty(8, 64, device="cuda"),
                torch.empty(64, 8, dtype=torch.bfloat16, device="cuda").t(), torch.empty(1, 64, dtype=torch.bfloat16, device="cuda").expand(8, 64)):
        with pytest.raises(ValueError, match="out must"):
            f(A, W, off, out=out)
    with pytest.raises(ValueError, match="overlaps"):
        f(A, W, off, out=A)


def test_a_group_of_almost_2_31_rows():
    """Rows and tiles of one group together pass 2^31: the tile's height must not wrap round."""
    from llm_reproducibility_b200.tbik.grouped_matmul import grouped_matmul_tp_persistent
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("needs 60 GB")
    M, K, period = 2 ** 31 - 300, 8, 4096
    some = make((period, K), torch.bfloat16, "int", 1)
    A = some.repeat(M // period + 1, 1)[:M]
    W = make((2, 1, K), torch.bfloat16, "int", 2)
    C = grouped_matmul_tp_persistent(A, W, torch.tensor([0, 5, M], dtype=torch.int32, device="cuda")).flatten()
    first, rest = ((some.double() @ W[g, 0].double()).to(torch.bfloat16) for g in range(2))
    assert torch.equal(C[:5], first[:5]) and torch.equal(C[5:period], rest[5:])
    whole = M // period * period
    assert (C[period:whole].view(-1, period) == rest).all() and torch.equal(C[whole:], rest[:M - whole])
    del A, C
    torch.cuda.empty_cache()
