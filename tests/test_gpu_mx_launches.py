"""The launch counter counts the kernels that the microscaled operators launch: those of a captured graph."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


def _kernels(graph) -> int:
    from cuda.bindings import runtime

    raw = graph.raw_cuda_graph()
    err, _, count = runtime.cudaGraphGetNodes(raw, 0)
    assert err == runtime.cudaError_t.cudaSuccess
    err, nodes, count = runtime.cudaGraphGetNodes(raw, count)
    kinds = [runtime.cudaGraphNodeGetType(n)[1] for n in nodes[:count]]
    return sum(k == runtime.cudaGraphNodeType.cudaGraphNodeTypeKernel for k in kinds)


def _check(call):
    from dimq_b200 import _lib

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        call()
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(g):
        before = _lib.LAUNCH_COUNT[0]
        keep = call()
        count = _lib.LAUNCH_COUNT[0] - before
    assert count == _kernels(g)
    del keep
    return count


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("m,k,n", [(1, 64, 32), (20, 64, 31), (300, 96, 72), (2000, 64, 72), (300, 600, 5000)])
def test_launch_counter(cuda_device, m, k, n, dtype):
    from dimq_b200 import ops, qat

    x, w, dy = torch.randn(m, k, device="cuda").to(dtype), torch.randn(n, k, device="cuda"), torch.randn(m, n, device="cuda").to(dtype)
    b = torch.randn(n, device="cuda")
    q, kept = ops.mx_quantize(w), ops.mx_quantize(x, "int8")
    assert _check(lambda: ops.mx_quantize(x)) == 1
    _check(lambda: ops.mx_dequantize(*kept, k, "int8"))
    _check(lambda: ops.mx_linear(x, *q, b, n, k))
    _check(lambda: ops.mx_linear_grad_input(dy, *q, k))
    _check(lambda: ops.mx_linear_grad_weight(dy, *kept, k))
    for keep in ("int8", "fp4"):
        for grads in ((True, True, True), (True, False, False), (False, True, True), (False, False, True), (False, False, False)):
            leaves = [t.clone().requires_grad_(g) for t, g in zip((x, w, b), grads)]
            need = [t for t in leaves if t.requires_grad]

            def step():
                y = qat.mx_linear(*leaves, checkpoint=keep)
                return torch.autograd.grad(y, need, dy) if need else y

            _check(step)
    x.requires_grad_(), b.requires_grad_()
    _check(lambda: torch.autograd.grad(ops.mx_linear(x, *q, b, n, k, out_dtype=dtype), (x, b), dy))
