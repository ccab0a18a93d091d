"""Low-rank adapters of many requests against a 64-bit restatement: bit for bit on small integers (every sum exact in any
order, h below 2^16), within a derived bound on normal deviates."""
import pytest
import torch

pytestmark = pytest.mark.gpu

HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def make(shape, dtype, kind, seed, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    if kind == "int":
        return torch.randint(-1, 2, shape, generator=g, device="cuda").to(dtype)
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def case(T, L, R, K, N, dtype, kind, seed=0, none=0.2):
    g = torch.Generator().manual_seed(seed + T)
    ids = torch.randint(0, L, (T,), generator=g)
    ids[torch.rand(T, generator=g) < none] = -1
    scales = torch.full((L,), 2.0) if kind == "int" else torch.rand(L, generator=g) + 0.5
    return (make((T, N), dtype, kind, seed + 1), make((T, K), dtype, kind, seed + 2), make((L, R, K), dtype, kind, seed + 3, K ** -0.5),
            make((L, N, R), dtype, kind, seed + 4, 0.3), ids.to(torch.int32).cuda(), scales.cuda())


def ref(y, x, A, B, ids, scales):
    """(out, h, bound of the fp32 work) in fp64."""
    out, size = y.double(), torch.zeros(y.shape, dtype=torch.float64, device=y.device)
    h = torch.zeros(y.shape[0], A.shape[1], dtype=torch.float64, device=y.device)
    K, R = A.shape[2], A.shape[1]
    for a in range(A.shape[0]):
        rows = torch.nonzero(ids == a).flatten()
        xa, Aa, Ba, s = x[rows].double(), A[a].double(), B[a].double(), float(scales[a])
        h[rows] = xa @ Aa.t()
        out[rows] += s * (h[rows] @ Ba.t())
        # h: K terms, each addition off by at most 2^-23 of the magnitudes; the second product reads h in two parts of the
        # operand type (off by 2^-16 of h at most) and adds R terms; scale and y: three more roundings
        mag = (xa.abs() @ Aa.abs().t()) * K * 2.0 ** -23 + h[rows].abs() * (2.0 ** -16 + (2 * R + 3) * 2.0 ** -23)
        size[rows] = s * (mag @ Ba.abs().t()) + y[rows].double().abs() * 2.0 ** -22
    return out, h, size


def check(got, want, kind):
    out, _, size = want
    if kind == "int":
        assert torch.equal(got, out.to(got.dtype)), (got.double() - out).abs().max()
    else:
        tol = HALF[got.dtype] * out.abs() + size * (1 + HALF[got.dtype]) + 2.0 ** -25
        bad = (got.double() - out).abs() > tol
        assert not bad.any(), (int(bad.sum()), ((got.double() - out).abs() - tol).max())


SHAPES = [(1, 1, 8, 8, 8), (1, 16, 16, 4096, 4096), (3, 2, 64, 40, 24), (16, 5, 16, 256, 264), (17, 1, 32, 1000, 72), (65, 64, 8, 520, 1032),
          (96, 48, 16, 2056, 512), (130, 3, 128, 776, 136), (300, 7, 24, 12288, 256), (33, 1024, 40, 264, 520), (2000, 4, 32, 512, 1024),
          (4500, 9, 72, 136, 328)]


@pytest.mark.parametrize("kind", ["int", "normal"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,L,R,K,N", SHAPES)
def test_lora_add(T, L, R, K, N, dtype, kind):
    from llm_reproducibility_b200.tbik.adapters import lora_add
    from llm_reproducibility_b200.tbik.row_groups import group_rows
    y, x, A, B, ids, s = case(T, L, R, K, N, dtype, kind)
    want = ref(y, x, A, B, ids, s)
    groups = group_rows(ids, L)
    keep = y.clone()
    got = lora_add(y, x, A, B, groups, s)
    check(got, want, kind)
    assert torch.equal(y, keep) and torch.equal(got[ids < 0], y[ids < 0])  # rows without adapter: their bits
    assert lora_add(y, x, A, B, groups, s, out=y) is y
    assert torch.equal(y, got)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,L,R,K,N", [(5, 3, 16, 512, 64), (200, 6, 32, 4096, 264), (1, 1, 8, 264, 8), (1500, 2, 128, 1024, 200)])
def test_shrink_and_expand_are_the_two_halves(T, L, R, K, N, dtype):
    from llm_reproducibility_b200.tbik.adapters import lora_add, lora_expand_add, lora_shrink
    from llm_reproducibility_b200.tbik.row_groups import group_rows
    y, x, A, B, ids, s = case(T, L, R, K, N, dtype, "normal")
    groups = group_rows(ids, L)
    h = lora_shrink(x, A, groups)
    want = ref(y, x, A, B, ids, s)[1]
    assert h.dtype == torch.float32 and (h[ids < 0] == 0).all()
    bound = sum(torch.where((ids == a)[:, None], x.double().abs() @ A[a].double().abs().t(), 0.0) for a in range(L)) * (K + 8) * 2.0 ** -23
    assert ((h.double() - want).abs() <= bound + 2.0 ** -40).all()
    assert torch.equal(lora_expand_add(y, h, B, groups, s), lora_add(y, x, A, B, groups, s))


@pytest.mark.parametrize("T", [5, 700])
def test_the_halves_do_not_read_the_width_that_they_have_no_part_in(T):
    """Through the C ABI, where a caller may pass any: the same bits."""
    from llm_reproducibility_b200 import _lib
    from llm_reproducibility_b200.tbik.adapters import lora_expand_add, lora_shrink
    from llm_reproducibility_b200.tbik.row_groups import group_rows
    y, x, A, B, ids, s = case(T, 3, 16, 520, 264, torch.bfloat16, "normal")
    g = group_rows(ids, 3)
    stream = torch.cuda.current_stream().cuda_stream
    want = lora_shrink(x, A, g)
    for N in (8, 4096, (1 << 24) - 8):
        h = torch.empty_like(want)
        assert _lib.lib().tbik_adapters(x.data_ptr(), 520, 0, 0, 0, 0, A.data_ptr(), 0, 0, h.data_ptr(), g.order.data_ptr(),
                                        g.offsets.data_ptr(), T, N, 520, 16, 3, 0, 0, stream) == 0
        assert torch.equal(h, want)
    want = lora_expand_add(y, h, B, g, s)
    for K in (8, 4096, (1 << 24) - 8):
        out = torch.empty_like(y)
        assert _lib.lib().tbik_adapters(0, 0, y.data_ptr(), 264, out.data_ptr(), 264, 0, B.data_ptr(), s.data_ptr(), h.data_ptr(),
                                        g.order.data_ptr(), g.offsets.data_ptr(), T, 264, K, 16, 3, 0, 0, stream) == 0
        assert torch.equal(out, want)


@pytest.mark.parametrize("K,tp", [(4096, 2), (4096, 8), (768, 4), (256, 8)])
def test_shards_of_k_add_up_to_the_unsharded_bits(K, tp):
    from llm_reproducibility_b200.tbik.adapters import leaf_for_adapters, lora_shrink
    from llm_reproducibility_b200.tbik.row_groups import group_rows
    _, x, A, _, ids, _ = case(77, 5, 16, K, 8, torch.bfloat16, "normal")
    groups, leaf, ks = group_rows(ids, 5), leaf_for_adapters(K, tp), K // tp
    parts = [lora_shrink(x[:, r * ks:(r + 1) * ks], A[:, :, r * ks:(r + 1) * ks], groups, leaf=leaf) for r in range(tp)]
    while len(parts) > 1:
        parts = [parts[i] + parts[i + 1] for i in range(0, len(parts), 2)]
    assert torch.equal(parts[0], lora_shrink(x, A, groups))


@pytest.mark.parametrize("R", [8, 128])
@pytest.mark.parametrize("T", [1, 40, 1500])
def test_a_leaf_wider_than_k_is_one_leaf_of_all_k(T, R):
    from llm_reproducibility_b200.tbik.adapters import lora_add
    from llm_reproducibility_b200.tbik.row_groups import group_rows
    K = 1000
    y, x, A, B, ids, s = case(T, 3, R, K, 72, torch.bfloat16, "int")
    groups, want = group_rows(ids, 3), ref(y, x, A, B, ids, s)[0].to(torch.bfloat16)
    for leaf in (1024, 1 << 20, 1 << 28, (1 << 31) - 32, 1 << 40):
        assert torch.equal(lora_add(y, x, A, B, groups, s, leaf=leaf), want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("R", [8, 16, 24, 32, 40, 64, 128])
def test_a_row_has_the_same_bits_in_every_batch(R, dtype):
    """One row, a decode batch, prompts: tiles and their work differ, the bits do not."""
    from llm_reproducibility_b200.tbik.adapters import lora_add
    from llm_reproducibility_b200.tbik.row_groups import group_rows
    y, x, A, B, ids, s = case(3000, 6, R, 1032, 328, dtype, "normal", none=0.1)
    full = lora_add(y, x, A, B, group_rows(ids, 6), s)
    for rows in (slice(0, 1), slice(5, 9), slice(100, 140), slice(500, 1524), slice(700, 1725)):
        part = lora_add(y[rows], x[rows], A, B, group_rows(ids[rows], 6), s)
        assert torch.equal(part, full[rows])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,L,R", [(96, 48, 32), (96, 48, 64), (96, 48, 128), (64, 1000, 64), (256, 1000, 16), (500, 1000, 32), (1000, 48, 16), (300, 4, 128)])
def test_few_rows_of_many_adapters_and_of_large_ranks(T, L, R, dtype):
    """Batches on either side of where tiles come through shared memory: the definition's values, and each row's bits alone."""
    from llm_reproducibility_b200.tbik.adapters import lora_add
    from llm_reproducibility_b200.tbik.row_groups import group_rows
    y, x, A, B, ids, s = case(T, L, R, 1032, 264, dtype, "normal")
    full = lora_add(y, x, A, B, group_rows(ids, L), s)
    check(full, ref(y, x, A, B, ids, s), "normal")
    for t in (0, T // 3, T - 1):
        assert torch.equal(lora_add(y[t:t + 1], x[t:t + 1], A, B, group_rows(ids[t:t + 1], L), s), full[t:t + 1])


def test_values_beyond_the_operand_types_range_in_h():
    """h is held in 32 bits: it may pass fp16's largest number."""
    from llm_reproducibility_b200.tbik.adapters import lora_add
    from llm_reproducibility_b200.tbik.row_groups import group_rows
    T, K, N, R = 20, 1024, 64, 16
    x, A = torch.full((T, K), 16.0, dtype=torch.float16, device="cuda"), torch.full((1, R, K), 16.0, dtype=torch.float16, device="cuda")
    B = torch.full((1, N, R), 2.0 ** -14, dtype=torch.float16, device="cuda")
    A[:, 1] = -16.0
    B[:, :, 3] = 0.0
    y = torch.ones((T, N), dtype=torch.float16, device="cuda")
    got = lora_add(y, x, A, B, group_rows(torch.zeros(T, dtype=torch.int32, device="cuda"), 1), torch.ones(1, device="cuda"))
    assert torch.equal(got, torch.full_like(got, 1 + (R - 3) * 2.0 ** 18 * 2.0 ** -14))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("R", [8, 16, 24, 32, 64, 128])
@pytest.mark.parametrize("T", [1, 40, 1500])
def test_h_is_multiplied_with_all_its_bits(T, R, dtype):
    """What is left where y and the adapter's terms cancel: the last bits of h."""
    from llm_reproducibility_b200.tbik.adapters import lora_expand_add
    from llm_reproducibility_b200.tbik.row_groups import group_rows
    g, N = torch.Generator(device="cuda").manual_seed(R), 72
    groups, one = group_rows(torch.zeros(T, dtype=torch.int32, device="cuda"), 1), torch.ones(1, device="cuda")
    # h against itself without its last five bits, through entries of 1: the sum of the two is those bits, exactly
    h = torch.randn(T, R, generator=g, device="cuda") + 3.0
    cut = (h.view(torch.int32) & -32).view(torch.float32)
    B = torch.zeros(1, N, R, dtype=dtype, device="cuda")
    for n in range(N):
        B[0, n, n % R] = B[0, n, (n + 1) % R] = 1.0
    pair = torch.where(torch.arange(R, device="cuda") % 2 == 0, h, -cut.roll(1, 1))
    want = torch.stack([pair[:, n % R].double() + pair[:, (n + 1) % R].double() for n in range(N)], 1)
    got = lora_expand_add(torch.zeros(T, N, dtype=dtype, device="cuda"), pair, B, groups, one)
    even = torch.arange(N, device="cuda") % R % 2 == 0
    assert want[:, even].abs().max() < 2.0 ** -16 and want[:, even].abs().max() > 0
    # (fp16: below its smallest normal number a result is off by half of its smallest step, 2^-25, at most)
    assert ((got.double() - want)[:, even].abs() <= HALF[dtype] * want[:, even].abs() + 2.0 ** -25 * (dtype == torch.float16)).all()
    # any entries, y the rounded opposite of the adapter's term: R products of three parts and one sum with y, each addition off by at
    # most 2^-23 of the magnitudes, then the rounding of the result
    B, s = (torch.randn(1, N, R, generator=g, device="cuda") * 0.3).to(dtype), torch.tensor([0.75], device="cuda")
    term, size = 0.75 * (h.double() @ B[0].double().t()), 0.75 * (h.double().abs() @ B[0].double().abs().t())
    y = (-term).to(dtype)
    want = y.double() + term
    tol = HALF[dtype] * want.abs() + ((3 * R + 3) * size + 2 * y.double().abs()) * 2.0 ** -23 + 2.0 ** -25
    assert ((lora_expand_add(y, h, B, groups, s).double() - want).abs() <= tol).all()


@pytest.mark.parametrize("R", [8, 32, 64])
@pytest.mark.parametrize("T", [1, 40, 1500])
def test_h_beyond_the_operand_types_largest_number(T, R):
    from llm_reproducibility_b200.tbik.adapters import lora_expand_add
    from llm_reproducibility_b200.tbik.row_groups import group_rows
    groups, one = group_rows(torch.zeros(T, dtype=torch.int32, device="cuda"), 1), torch.ones(1, device="cuda")
    # bf16: fp32's largest number, which rounds to bf16's infinity; fp16: 2^120, of either sign, against bits of 2^-14
    for dtype, big, small in ((torch.bfloat16, torch.finfo(torch.float32).max, 2.0 ** -120), (torch.float16, 2.0 ** 120, 2.0 ** -14)):
        h, B = torch.zeros(T, R, device="cuda"), torch.zeros(1, 72, R, dtype=dtype, device="cuda")
        h[:, 1], h[:, 5], B[0, :, 5] = big, -big, small
        B[0, ::2, 1] = small
        want = h.double() @ B[0].double().t()
        got = lora_expand_add(torch.zeros(T, 72, dtype=dtype, device="cuda"), h, B, groups, one)
        assert torch.equal(got, want.to(dtype)) and (got[:, ::2] == 0).all()


def test_infinities_and_nan_stay_in_their_rows():
    from llm_reproducibility_b200.tbik.adapters import lora_add
    from llm_reproducibility_b200.tbik.row_groups import group_rows
    for bad in (float("nan"), float("inf")):
        y, x, A, B, ids, s = case(70, 3, 16, 512, 128, torch.bfloat16, "int", none=0.0)
        want = ref(y, x, A, B, ids, s)[0].to(torch.bfloat16)
        x[9] = bad
        A[2, 5], B[2, 7] = bad, bad
        got = lora_add(y, x, A, B, group_rows(ids, 3), s)
        fine = [t for t in range(70) if t != 9 and int(ids[t]) != 2]
        assert torch.equal(got[fine], want[fine]) and not got[9].isfinite().all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("R", [8, 16, 24, 32, 64, 128])
@pytest.mark.parametrize("K,leaf", [(9224, None), (1000, 1024), (5000, 5024), (12288, 4096)])
def test_a_leaf_in_several_pieces_has_the_bits_of_a_leaf_in_one(K, leaf, R, dtype):
    """Few rows bring a leaf to shared memory in pieces whose width goes by the rank and the rows of the tile; many rows walk it."""
    from llm_reproducibility_b200.tbik.adapters import lora_add, lora_shrink
    from llm_reproducibility_b200.tbik.row_groups import group_rows
    y, x, A, B, ids, s = case(1100, 5, R, K, 72, dtype, "normal", none=0.1)
    groups = group_rows(ids, 5)
    full, h = lora_add(y, x, A, B, groups, s, leaf=leaf), lora_shrink(x, A, groups, leaf=leaf)
    for rows in (slice(0, 1), slice(5, 9), slice(100, 140), slice(400, 900)):
        part = group_rows(ids[rows], 5)
        assert torch.equal(lora_shrink(x[rows], A, part, leaf=leaf), h[rows])
        assert torch.equal(lora_add(y[rows], x[rows], A, B, part, s, leaf=leaf), full[rows])
    check(full, ref(y, x, A, B, ids, s), "normal")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kind", ["int", "normal"])
@pytest.mark.parametrize("R", [8, 16, 24, 32, 64])
@pytest.mark.parametrize("T", [1, 40, 1500])
def test_an_infinite_entry_of_b_gives_what_the_sum_gives(T, R, kind, dtype):
    """+-inf where h is not zero there, NaN where it is or where two infinities meet with both signs; nothing else moves."""
    from llm_reproducibility_b200.tbik.adapters import lora_add
    from llm_reproducibility_b200.tbik.row_groups import group_rows
    inf = float("inf")
    y, x, A, B, ids, s = case(T, 2, R, 64, 72, dtype, kind, none=0.0)
    x[:, :16] = 0                     # rows 3 and 4 of A see nothing else: h = 0 there
    A[:, 3:5, 16:] = 0
    clean = lora_add(y, x, A, B, group_rows(ids, 2), s)
    B[0, 5, 1], B[0, 6, 3], B[1, 9, 2], B[1, 9, R - 1], B[1, 70, 0] = inf, -inf, -inf, inf, inf
    groups, (want, _, size) = group_rows(ids, 2), ref(y, x, A, B, ids, s)
    got = lora_add(y, x, A, B, groups, s)
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.isinf(), want.isinf())
    assert torch.equal(got[got.isinf()].double(), want[want.isinf()])
    assert torch.equal(got[want.isfinite()], clean[want.isfinite()])
    if T > 1:
        assert want.isnan().any() and want.isinf().any()
    assert torch.equal(lora_add(y, x, A, B, groups, s, out=y).nan_to_num(0.0, 1.0, -1.0), got.nan_to_num(0.0, 1.0, -1.0))


def test_no_adapters_at_all_and_no_rows():
    from llm_reproducibility_b200.tbik.adapters import lora_add, lora_shrink
    from llm_reproducibility_b200.tbik.row_groups import group_rows
    y, x, A, B, ids, s = case(50, 4, 16, 64, 72, torch.bfloat16, "normal", none=1.1)
    groups = group_rows(ids, 4)
    assert torch.equal(lora_add(y, x, A, B, groups, s), y)
    assert (lora_shrink(x, A, groups) == 0).all()
    empty = group_rows(ids[:0], 4)
    assert lora_add(y[:0], x[:0], A, B, empty, s).shape == (0, 72)


def test_strides_and_neighbours():
    from llm_reproducibility_b200.tbik.adapters import lora_add
    from llm_reproducibility_b200.tbik.row_groups import group_rows
    T, K, N = 37, 64, 72
    y, x, A, B, ids, s = case(T, 3, 16, K, N, torch.bfloat16, "int")
    groups, want = group_rows(ids, 3), ref(y, x, A, B, ids, s)[0].to(torch.bfloat16)
    wx = torch.zeros(T, 3 * K + 3, dtype=torch.bfloat16, device="cuda")
    for view in (wx[:, :K], wx[:, 1:K + 1], wx[:, ::3][:, :K]):
        view.copy_(x)
        assert torch.equal(lora_add(y, view, A, B, groups, s), want)
    assert torch.equal(lora_add(y, x, A.transpose(1, 2).contiguous().transpose(1, 2), B.transpose(1, 2).contiguous().transpose(1, 2), groups, s), want)
    buf = torch.full((T + 2, N + 16), 9.0, dtype=torch.bfloat16, device="cuda")
    lora_add(y, x, A, B, groups, s, out=buf[1:T + 1, 8:8 + N])
    assert torch.equal(buf[1:T + 1, 8:8 + N], want)
    buf[1:T + 1, 8:8 + N] = 9.0
    assert (buf == 9.0).all()
    # one row for all: a broadcast x
    same = x[:1].expand(T, K)
    assert torch.equal(lora_add(y, same, A, B, groups, s), ref(y, same, A, B, ids, s)[0].to(torch.bfloat16))


def test_x_and_the_result_are_columns_of_one_buffer():
    from llm_reproducibility_b200.tbik.adapters import lora_add
    from llm_reproducibility_b200.tbik.row_groups import group_rows
    T, K, N = 37, 64, 72
    y, x, A, B, ids, s = case(T, 3, 16, K, N, torch.bfloat16, "int")
    groups, want = group_rows(ids, 3), ref(y, x, A, B, ids, s)[0].to(torch.bfloat16)
    for at_x, at_y in ((0, K), (N, 0)):
        buf = torch.zeros(T, K + N, dtype=torch.bfloat16, device="cuda")
        vx, vy = buf[:, at_x:at_x + K].copy_(x), buf[:, at_y:at_y + N].copy_(y)
        assert lora_add(vy, vx, A, B, groups, s, out=vy) is vy and torch.equal(vy, want) and torch.equal(vx, x)
        with pytest.raises(ValueError, match="overlaps"):
            lora_add(y, vx, A, B, groups, s, out=buf[:, 8:8 + N])


def test_one_row_of_a_buffer_with_an_odd_pitch():
    """The stride between the rows of a single row is never stepped and says nothing: not of x, y, h, nor of out."""
    from llm_reproducibility_b200.tbik.adapters import lora_add, lora_expand_add, lora_shrink
    from llm_reproducibility_b200.tbik.row_groups import group_rows
    K, N, R = 64, 72, 16
    for ids in (torch.zeros(1, dtype=torch.int32, device="cuda"), torch.full((1,), -1, dtype=torch.int32, device="cuda")):
        y, x, A, B, _, s = case(1, 3, R, K, N, torch.bfloat16, "int")
        groups, (want, h, _) = group_rows(ids, 3), ref(y, x, A, B, ids, s)
        want = want.to(torch.bfloat16)
        wide = lambda t, pitch: torch.zeros(4, pitch, dtype=t.dtype, device="cuda")[:1, :t.shape[1]].copy_(t)  # noqa: E731
        for px, py in ((K + 3, N + 3), (K, N + 1), (K + 5, N + 8)):
            wx, wy, wh = wide(x, px), wide(y, py), wide(h.float(), R + 3)
            assert torch.equal(lora_shrink(wx, A, groups).double(), h)
            for f in (lambda **kw: lora_add(wy, wx, A, B, groups, s, **kw), lambda **kw: lora_expand_add(wy, wh, B, groups, s, **kw)):
                assert torch.equal(f(), want) and torch.equal(wy, y)
                buf = torch.full((3, N + 11), 9.0, dtype=torch.bfloat16, device="cuda")
                assert torch.equal(f(out=buf[:1, :N]), want) and (buf[1:] == 9).all() and (buf[:, N:] == 9).all()
                again = wy.as_strided((1, N), (N, 1))  # the same row, said otherwise
                assert torch.equal(f(out=again), want) and torch.equal(wy, want)
                wy.copy_(y)


def test_bad_tables_touch_nothing_outside():
    from llm_reproducibility_b200.tbik.adapters import lora_add
    from llm_reproducibility_b200.tbik.row_groups import RowGroups
    T, K, N = 40, 64, 64
    y, x, A, B, ids, s = case(T, 3, 16, K, N, torch.bfloat16, "int")
    buf = torch.full((T + 2, N), 9.0, dtype=torch.bfloat16, device="cuda")
    for order, offsets in (([2 ** 31 - 1] * T, [0, 10, 20, 40]), ([-1] * T, [0, 10, 20, 40]), (list(range(T)), [0, 1000, 2000, 2 ** 31 - 1]),
                           (list(range(T)), [-7, 30, 10, 50]), (list(range(T)), [2 ** 31 - 1, 0, 0, 0])):
        g = RowGroups(torch.tensor(order, dtype=torch.int32, device="cuda"), None, torch.tensor(offsets, dtype=torch.int32, device="cuda"))
        lora_add(y, x, A, B, g, s, out=buf[1:T + 1])
        assert (buf[0] == 9).all() and (buf[-1] == 9).all()


def test_streams_and_a_graph_that_follows_new_ids():
    from llm_reproducibility_b200.tbik.adapters import lora_add
    from llm_reproducibility_b200.tbik.row_groups import group_rows
    y, x, A, B, ids, s = case(64, 5, 16, 512, 256, torch.bfloat16, "int")
    lora_add(y, x, A, B, group_rows(ids, 5), s)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = lora_add(y, x, A, B, group_rows(ids, 5), s)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, ref(y, x, A, B, ids, s)[0].to(torch.bfloat16))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = lora_add(y, x, A, B, group_rows(ids, 5), s)
    for shift in (1, 2):
        ids.copy_((torch.arange(64, device="cuda") * shift) % 7 - 1)
        graph.replay()
        assert torch.equal(out, ref(y, x, A, B, torch.where(ids < 5, ids, -1), s)[0].to(torch.bfloat16))


def test_rows_beyond_32_bit_offsets():
    """More than 2^31 elements in y: rows at the end of a long batch."""
    from llm_reproducibility_b200.tbik.adapters import lora_add
    from llm_reproducibility_b200.tbik.row_groups import group_rows
    T, N, K, R = 140000, 16384, 64, 16
    ids = (torch.arange(T, device="cuda") % 3 - 1).to(torch.int32)
    x, A, B = make((T, K), torch.bfloat16, "int", 1), make((2, R, K), torch.bfloat16, "int", 2), make((2, N, R), torch.bfloat16, "int", 3)
    y = torch.ones(T, N, dtype=torch.bfloat16, device="cuda")
    assert y.numel() > 1 << 31
    s = torch.tensor([1.0, 2.0], device="cuda")
    lora_add(y, x, A, B, group_rows(ids, 2), s, out=y)
    for rows in (slice(0, 50), slice(131060, 131100), slice(T - 50, T)):
        want = ref(torch.ones(rows.stop - rows.start, N, dtype=torch.bfloat16, device="cuda"), x[rows], A, B, ids[rows], s)[0]
        assert torch.equal(y[rows], want.to(torch.bfloat16))


def test_refusals_on_the_device():
    from llm_reproducibility_b200.tbik.adapters import lora_add
    from llm_reproducibility_b200.tbik.row_groups import group_rows
    y, x, A, B, ids, s = case(20, 3, 16, 64, 64, torch.bfloat16, "int")
    g = group_rows(ids, 3)
    buf = torch.zeros(21, 64, dtype=torch.bfloat16, device="cuda")
    for bad_y, out in ((y, x), (buf[:20], buf[1:]), (y, torch.empty(20, 64, device="cuda")), (y, torch.empty(20, 68, dtype=torch.bfloat16, device="cuda")[:, 4:])):
        with pytest.raises(ValueError, match="out"):
            lora_add(bad_y, x, A, B, g, s, out=out)
    with pytest.raises(RuntimeError, match="CUDA"):
        lora_add(y, x, A, B, g, s.cpu())
    with pytest.raises(ValueError, match="offsets"):
        lora_add(y, x, A, B, group_rows(ids, 4), s)
