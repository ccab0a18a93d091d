"""What the grouped operators refuse, through the Python entry points and through the C ABI, without a GPU: every check
stands before the first launch."""
import pytest
import torch

BF16 = torch.bfloat16


def off(*values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype)


def test_grouped_matmul_refuses():
    from llm_reproducibility_b200.tbik.grouped_matmul import grouped_matmul_tp_persistent as f
    A, W = torch.zeros(4, 128, dtype=BF16), torch.zeros(2, 8, 128, dtype=BF16)
    with pytest.raises(RuntimeError, match="CUDA"):
        f(A, W, off(0, 2, 4))
    with pytest.raises(ValueError, match="A must be"):
        f(A, W[0], off(0, 2, 4))
    with pytest.raises(ValueError, match="A must be"):
        f(A[:, :64], W, off(0, 2, 4))
    with pytest.raises(NotImplementedError):
        f(A.float(), W.float(), off(0, 2, 4))
    with pytest.raises(ValueError, match="operands"):
        f(A, W.half(), off(0, 2, 4))
    with pytest.raises(ValueError, match="int32"):
        f(A, W, off(0, 2, 4, dtype=torch.int64))
    with pytest.raises(ValueError, match="3 entries"):
        f(A, W, off(0, 4))
    for leaf in (0, 32, 96, 256, -64):
        with pytest.raises(ValueError, match="leaf"):
            f(A, W, off(0, 2, 4), leaf=leaf)
    with pytest.raises(ValueError, match="out_dtype"):
        f(A, W, off(0, 2, 4), out_dtype=torch.float64)
    with pytest.raises(ValueError, match="groups"):
        f(A, torch.zeros(1025, 8, 128, dtype=BF16), torch.zeros(1026, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="tree_grouped_linear"):
        f(A.clone().requires_grad_(True), W, off(0, 2, 4))
    with torch.no_grad(), pytest.raises(RuntimeError, match="CUDA"):
        f(A.clone().requires_grad_(True), W, off(0, 2, 4))


def test_weight_gradient_refuses():
    from llm_reproducibility_b200.tbik.grouped_matmul import grouped_weight_gradient as f
    A, D = torch.zeros(4, 16, dtype=BF16), torch.zeros(4, 8, dtype=BF16)
    with pytest.raises(RuntimeError, match="CUDA"):
        f(D, A, off(0, 2, 4))
    with pytest.raises(ValueError, match="dC must be"):
        f(D[:3], A, off(0, 2, 4))
    with pytest.raises(ValueError, match="groups"):
        f(D, A, off(0))
    with pytest.raises(ValueError, match="int32"):
        f(D, A, off(0, 4, dtype=torch.int64))
    with pytest.raises(ValueError, match="operands"):
        f(D.half(), A, off(0, 4))


def test_router_refuses():
    from llm_reproducibility_b200.tbik.autograd import tree_route_topk
    from llm_reproducibility_b200.tbik.row_groups import group_rows, route_topk
    x = torch.zeros(4, 8)
    for f in (route_topk, tree_route_topk):
        with pytest.raises(RuntimeError, match="CUDA"):
            f(x, 2)
        with pytest.raises(ValueError, match="k must"):
            f(x, 9)
        with pytest.raises(ValueError, match="k must"):
            f(x, 0)
        with pytest.raises(ValueError, match="tokens, experts"):
            f(x[0], 2)
        with pytest.raises(NotImplementedError):
            f(x.double(), 2)
        with pytest.raises(ValueError, match="experts must"):
            f(torch.zeros(2, 1025), 2)
        with pytest.raises(ValueError, match="k must"):
            f(torch.zeros(2, 100), 33)
    with pytest.raises(RuntimeError, match="tree_route_topk"):
        route_topk(x.clone().requires_grad_(True), 2)
    with pytest.raises(ValueError, match="int32"):
        group_rows(torch.zeros(4, dtype=torch.int64), 2)
    for n in (0, -1, 1025):
        with pytest.raises(ValueError, match="groups"):
            group_rows(torch.zeros(4, dtype=torch.int32), n)
    with pytest.raises(RuntimeError, match="CUDA"):
        group_rows(torch.zeros(4, dtype=torch.int32), 2)


def test_adapters_refuse():
    from llm_reproducibility_b200.tbik.adapters import leaf_for_adapters, lora_add, lora_expand_add, lora_shrink
    from llm_reproducibility_b200.tbik.row_groups import RowGroups
    y, x = torch.zeros(4, 24, dtype=BF16), torch.zeros(4, 64, dtype=BF16)
    A, B, s = torch.zeros(3, 8, 64, dtype=BF16), torch.zeros(3, 24, 8, dtype=BF16), torch.ones(3)
    g = RowGroups(torch.arange(4, dtype=torch.int32), torch.arange(4, dtype=torch.int32), off(0, 1, 2, 4))
    with pytest.raises(RuntimeError, match="CUDA"):
        lora_add(y, x, A, B, g, s)
    with pytest.raises(RuntimeError, match="CUDA"):
        lora_shrink(x, A, g)
    with pytest.raises(RuntimeError, match="CUDA"):
        lora_expand_add(y, torch.zeros(4, 8), B, g, s)
    for bad in ((y, x, A[:2], B, g, s), (y, x[:, :32], A, B, g, s), (y[:3], x, A, B, g, s), (y[:, :16], x, A, B, g, s)):
        with pytest.raises(ValueError, match="lora_add: y"):
            lora_add(*bad)
    with pytest.raises(ValueError, match="scales"):
        lora_add(y, x, A, B, g, s[:2])
    with pytest.raises(ValueError, match="scales"):
        lora_add(y, x, A, B, g, s.half())
    with pytest.raises(ValueError, match="offsets"):
        lora_add(y, x, A, B, g._replace(offsets=off(0, 4)), s)
    with pytest.raises(ValueError, match="order"):
        lora_add(y, x, A, B, g._replace(order=g.order.long()), s)
    with pytest.raises(ValueError, match="rank"):
        lora_shrink(x, torch.zeros(3, 12, 64, dtype=BF16), g)
    with pytest.raises(ValueError, match="rank"):
        lora_shrink(x, torch.zeros(3, 136, 64, dtype=BF16), g)
    with pytest.raises(ValueError, match="multiples of 8"):
        lora_shrink(x[:, :60], A[:, :, :60], g)
    with pytest.raises(NotImplementedError):
        lora_shrink(x.float(), A.float(), g)
    for leaf in (16, 40, -32, 0):
        with pytest.raises(ValueError, match="leaf"):
            lora_shrink(x, A, g, leaf=leaf)
    with pytest.raises(ValueError, match="h must"):
        lora_expand_add(y, torch.zeros(4, 8, dtype=BF16), B, g, s)
    with pytest.raises(RuntimeError, match="no gradient"):
        lora_add(y, x.clone().requires_grad_(True), A, B, g, s)
    assert leaf_for_adapters(4096) == 512 and leaf_for_adapters(100, 1) == 32
    with pytest.raises(ValueError):
        leaf_for_adapters(100, 2)
    with pytest.raises(ValueError):
        leaf_for_adapters(4096, 3)


def test_a_result_tensor_that_requires_a_gradient_is_refused():
    """It would come back with its old graph.  Without recording the call goes on (to the check of the device)."""
    from llm_reproducibility_b200.tbik.adapters import lora_add, lora_expand_add
    from llm_reproducibility_b200.tbik.grouped_matmul import grouped_matmul_tp_persistent
    from llm_reproducibility_b200.tbik.row_groups import RowGroups
    g = RowGroups(torch.arange(4, dtype=torch.int32), torch.arange(4, dtype=torch.int32), off(0, 2, 4))
    x, A, B, s = torch.zeros(4, 64, dtype=BF16), torch.zeros(2, 8, 64, dtype=BF16), torch.zeros(2, 16, 8, dtype=BF16), torch.ones(2)
    leaf = torch.zeros(4, 16, dtype=BF16, requires_grad=True)
    for out in (leaf, leaf * 2, leaf[:, :]):
        for call in (lambda: grouped_matmul_tp_persistent(x, torch.zeros(2, 16, 64, dtype=BF16), g.offsets, out=out),
                     lambda: lora_add(torch.zeros(4, 16, dtype=BF16), x, A, B, g, s, out=out),
                     lambda: lora_expand_add(torch.zeros(4, 16, dtype=BF16), torch.zeros(4, 8), B, g, s, out=out)):
            with pytest.raises(RuntimeError, match="records no gradient"):
                call()
            with torch.no_grad(), pytest.raises(RuntimeError, match="CUDA"):
                call()


def test_forward_mode_tangents_are_refused():
    """A dual tensor does not require a gradient; its tangent must not be dropped without a word."""
    import torch.autograd.forward_ad as fwd
    from llm_reproducibility_b200.tbik.adapters import lora_add, lora_expand_add, lora_shrink
    from llm_reproducibility_b200.tbik.autograd import tree_grouped_linear, tree_route_topk
    from llm_reproducibility_b200.tbik.grouped_matmul import grouped_matmul_tp_persistent, grouped_weight_gradient
    from llm_reproducibility_b200.tbik.row_groups import RowGroups, route_topk
    g = RowGroups(torch.arange(4, dtype=torch.int32), torch.arange(4, dtype=torch.int32), off(0, 2, 4))
    x, A, B, s = torch.zeros(4, 64, dtype=BF16), torch.zeros(2, 8, 64, dtype=BF16), torch.zeros(2, 16, 8, dtype=BF16), torch.ones(2)
    y, h, W = torch.zeros(4, 16, dtype=BF16), torch.zeros(4, 8), torch.zeros(2, 16, 64, dtype=BF16)
    with fwd.dual_level():
        dual = lambda t: fwd.make_dual(t, torch.ones_like(t))  # noqa: E731
        for call in (lambda: route_topk(dual(x), 2), lambda: grouped_matmul_tp_persistent(dual(x), W, g.offsets),
                     lambda: grouped_matmul_tp_persistent(x, dual(W), g.offsets), lambda: grouped_matmul_tp_persistent(x, W, g.offsets, out=dual(y)),
                     lambda: grouped_weight_gradient(dual(y), x, g.offsets), lambda: lora_add(y, x, A, dual(B), g, s),
                     lambda: lora_add(y, x, A, B, g, dual(s)), lambda: lora_add(y, x, A, B, g, s, out=dual(y)),
                     lambda: lora_shrink(dual(x), A, g), lambda: lora_expand_add(y, dual(h), B, g, s)):
            with pytest.raises(RuntimeError, match="no tangent"):
                call()
            with torch.no_grad(), pytest.raises(RuntimeError, match="no tangent"):
                call()
        for call in (lambda: tree_grouped_linear(dual(x), W, g.offsets), lambda: tree_route_topk(dual(x), 2)):
            with pytest.raises(RuntimeError):  # (NotImplementedError is one: no jvp)
                call()
        with pytest.raises(RuntimeError, match="CUDA"):
            lora_shrink(x, A, g)


def test_widths_that_do_not_fit_the_kernels():
    """Broadcast operands may be wider than any memory: a width must not wrap round on its way to the kernel."""
    from llm_reproducibility_b200.tbik.adapters import lora_expand_add, lora_shrink
    from llm_reproducibility_b200.tbik.grouped_matmul import grouped_matmul_tp_persistent, grouped_weight_gradient
    from llm_reproducibility_b200.tbik.row_groups import RowGroups
    one = torch.zeros(1, dtype=BF16)
    g = RowGroups(torch.zeros(1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32), off(0, 1))
    for K in (1 << 24, (1 << 32) + 64):
        with pytest.raises(ValueError, match="2\\^24"):
            lora_shrink(one.expand(1, K), one.expand(1, 8, K), g)
        with pytest.raises(ValueError, match="2\\^24"):
            lora_expand_add(one.expand(1, K), torch.zeros(1, 8), one.expand(1, K, 8), g, torch.ones(1))
    for n in (1 << 30, (1 << 32) + 64):
        with pytest.raises(ValueError, match="2\\^30"):
            grouped_matmul_tp_persistent(one.expand(1, n), one.expand(1, 8, n), off(0, 1))
        with pytest.raises(ValueError, match="2\\^30"):
            grouped_matmul_tp_persistent(one.expand(1, 64), one.expand(1, n, 64), off(0, 1))
        with pytest.raises(ValueError, match="2\\^30"):
            grouped_weight_gradient(one.expand(1, n), one.expand(1, 8), off(0, 1))
        with pytest.raises(ValueError, match="2\\^30"):
            grouped_weight_gradient(one.expand(1, 8), one.expand(1, n), off(0, 1))


def test_c_abi_refuses_before_any_launch():
    from llm_reproducibility_b200 import _lib
    L = _lib.lib()
    p = 1 << 20  # a 16-byte aligned number that no check dereferences
    ok = [p, p, p, p, 4, 8, 128, 2, 128, 128, 1024, 8, 0, 0, 0, 0, 0, 0, None]

    def gemm(**at):
        args = list(ok)
        for i, v in at.items():
            args[int(i[1:])] = v
        return L.tbik_grouped_gemm(*args)

    assert gemm(_4=0) == 0 and gemm(_5=0) == 0                         # nothing to do
    assert gemm(_0=None) == -1 and gemm(_3=None) == -1 and gemm(_12=2) == -1
    assert gemm(_6=0) == -2 and gemm(_7=0) == -2 and gemm(_7=1025) == -2 and gemm(_4=1 << 31) == -2 and gemm(_15=48) == -2
    assert gemm(_8=120) == -2 and gemm(_9=64) == -2 and gemm(_10=512) == -2 and gemm(_11=4) == -2
    assert gemm(_13=2) == -3 and gemm(_14=1) == -3
    assert gemm(_0=p + 2) == -4 and gemm(_1=p + 8) == -4 and gemm(_8=129) == -4
    assert "tbik_grouped_gemm" in _lib.last_error()
    assert L.tbik_grouped_gemm_wgrad(p, p, None, p, 4, 8, 16, 2, 8, 16, 0, 0, 0, None) == -1
    assert L.tbik_grouped_gemm_wgrad(p, p, p, p, 4, 8, 16, 2, 4, 16, 0, 0, 0, None) == -2
    assert L.tbik_grouped_gemm_wgrad(p, p, p, p, 4, 8, 16, 2, 8, 17, 0, 0, 0, None) == -4
    assert L.tbik_grouped_gemm_wgrad(p, p, p, p, 4, 8, 16, 2, 8, 16, 0, 1, 0, None) == -3
    assert L.tbik_group_rows(p, 4, 0, p, p, p, p, 99, None) == -2 and L.tbik_group_rows(None, 4, 2, p, p, p, p, 99, None) == -1
    assert L.tbik_group_rows(p, 4, 2, p, p, None, p, 99, None) == -1 and L.tbik_group_rows(p, -1, 2, p, p, p, p, 99, None) == -2
    need = L.tbik_group_workspace_bytes(1 << 20, 128)
    assert need > 0 and L.tbik_group_rows(p, 1 << 20, 128, p, p, p, p, need - 1, None) == -1
    assert L.tbik_group_rows(p, 1 << 20, 128, p, p, p, None, need, None) == -1 and "workspace" in _lib.last_error()
    assert L.tbik_route_topk(p, 8, 4, 8, 2, 0, 1, p, p, p, p, p, None, 0, None) == -1
    assert L.tbik_route_topk(p, 8, 4, 8, 9, 0, 1, p, p, p, p, p, p, 999, None) == -2
    assert L.tbik_route_topk(p, 8, 4, 8, 2, 7, 1, p, p, p, p, p, p, 999, None) == -3
    assert L.tbik_route_topk(None, 8, 4, 8, 2, 0, 1, p, p, p, p, p, p, 999, None) == -1
    assert L.tbik_route_topk_backward(p, 8, 4, 8, 2, 0, 1, p, p, None, p, 8, None) == -1
    assert L.tbik_route_topk_backward(p, 8, 0, 8, 2, 0, 1, None, None, None, None, 8, None) == 0
    base = [p, 64, p, 24, p, 24, p, p, p, None, p, p, 4, 24, 64, 8, 3, 0, 0, None]

    def lora(**at):
        args = list(base)
        for i, v in at.items():
            args[int(i[1:])] = v
        return L.tbik_adapters(*args)

    assert lora(_12=0) == 0
    assert lora(_0=None) == -1 and lora(_2=None) == -1 and lora(_6=None) == -1 and lora(_10=None) == -1 and lora(_0=None, _2=None) == -1
    assert lora(_13=1 << 24, _3=1 << 24, _5=1 << 24) == -2 and lora(_14=1 << 24, _1=1 << 24) == -2
    assert lora(_13=20) == -2 and lora(_14=12) == -2 and lora(_15=12) == -2 and lora(_15=136) == -2 and lora(_16=0) == -2 and lora(_18=40) == -2
    assert lora(_1=32) == -2 and lora(_3=16) == -2 and lora(_17=2) == -3 and lora(_2=p + 4) == -4 and lora(_1=65) == -4


def test_c_abi_takes_groups_that_lie_row_by_row_in_turn():
    """[N, G, K] memory passes the strides' check (the next one, of the alignment, is what refuses here); strides at which
    groups meet do not."""
    from llm_reproducibility_b200 import _lib
    L, p = _lib.lib(), 1 << 20

    def gemm(ldw, stride_w, groups=4, N=8, K=128, layout=0):
        return L.tbik_grouped_gemm(p, p + 8, p, p, 4, N, K, groups, K, ldw, stride_w, N, layout, 0, 0, 0, 0, 0, None)

    assert gemm(128, 1024) == -4 and gemm(512, 128) == -4 and gemm(528, 128) == -4 and gemm(512, 64) == -2 and gemm(504, 128) == -2
    assert gemm(32, 8, layout=1) == -4 and gemm(24, 8, layout=1) == -2


def test_overlap_of_tensors():
    """Against the sets of bytes that two tensors touch: never false where they share one, true where only spans meet but for columns
    of one matrix."""
    from llm_reproducibility_b200.tbik.row_groups import overlap

    def touched(t):
        at = torch.arange(t.untyped_storage().nbytes() // t.element_size()).as_strided(t.shape, t.stride(), t.storage_offset())
        return {int(i) * t.element_size() + j for i in at.flatten() for j in range(t.element_size())}

    buf = torch.zeros(6, 40, dtype=BF16)
    flat = buf.view(-1)
    views = [buf, buf[:, :16], buf[:, 16:32], buf[:, 15:17], buf[2:, 32:], buf[:1], buf[1:2, :8], buf[:3, 8:24], buf[3:, 8:24], buf[:, ::2], buf[:0],
             buf[:, 5:5], flat[30:].as_strided((4, 20), (40, 1)), flat.as_strided((3, 16), (80, 1)), flat.as_strided((4, 30), (20, 1)), flat[20:60],
             buf.view(torch.float32)[:, 2:9], buf[1].expand(4, 40), buf.t()]
    for a in views:
        for b in views:
            assert overlap(a, b) or not (touched(a) & touched(b)), (a.shape, a.stride(), b.shape, b.stride())
    for a, b in ((buf[:, :16], buf[:, 16:32]), (buf[:, 16:32], buf[:, :16]), (buf[:, 8:16], buf[2:, 24:]), (buf[:3], buf[3:]), (buf[:, 0:1], buf[:, 39:])):
        assert not overlap(a, b)
