"""The dense product as the first CUDA call of a host thread: a backward pass runs in a thread of its own, and with the result
served from the allocator's cache nothing before the call has bound a context there."""
import threading

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_dense_product_from_a_new_thread():
    from llm_reproducibility_b200.tbik.tree_based_matmul import matmul_tp_persistent
    g = torch.Generator(device="cuda").manual_seed(1)
    A = torch.randn(64, 512, generator=g, device="cuda").to(torch.bfloat16)
    W = torch.randn(256, 512, generator=g, device="cuda").to(torch.bfloat16)
    spare = [torch.empty(64, 256, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    del spare
    torch.cuda.synchronize()
    got = []

    def work():
        try:
            got.append(matmul_tp_persistent(A, W.t()))
        except Exception as e:  # noqa: BLE001
            got.append(e)

    t = threading.Thread(target=work)
    t.start()
    t.join()
    torch.cuda.synchronize()
    assert torch.is_tensor(got[0]), got[0]
    assert torch.equal(got[0], matmul_tp_persistent(A, W.t()))
