"""Rows that lie in memory in their own way: products with 4-bit weights and the append to the 8-bit cache."""
import pytest
import torch

from cajeta_llm_b200.csrc import kernels as K
from test_gpu_q4 import DEV, F64, check, sums, weight

pytestmark = pytest.mark.gpu


def test_one_row_of_any_stride():
    """The stride of a single row says nothing: a column turned over is taken."""
    w, full = weight((200, 256), 64, seed=3)
    up, full_up = weight((3, 200, 256), 64, seed=4)
    x = torch.randn((256, 1), device=DEV).to(torch.bfloat16).t()
    assert x.stride(0) == 1
    out = torch.empty((1, 200), device=DEV)
    K.gemm_q4(x, w, out)
    xd = x.to(F64)
    check(out, xd @ full.T, sums(256, xd.abs() @ full.abs().T))
    # the same row for every row of a mixture, few and many
    for rows in (5, 40):
        out = torch.empty((rows, 200), device=DEV)
        edges = torch.tensor([0, 1, rows - 2, rows], dtype=torch.int32, device=DEV)
        K.gemm_q4(x, up, out, group_offsets=edges, a_row_index=torch.zeros(rows, dtype=torch.int32, device=DEV))
        for g in range(3):
            check(out[edges[g]:edges[g + 1]], (xd @ full_up[g].T).expand(int(edges[g + 1] - edges[g]), -1), sums(256, xd.abs() @ full_up[g].abs().T))


def test_one_row_of_any_stride_is_appended():
    heads, kv, hd, P = 2, 1, 64, 16
    x = torch.randn((4 * hd, 1), device=DEV).t()
    assert x.stride(0) == 1
    k, v = (torch.zeros((2, kv, P, hd), device=DEV).to(torch.float8_e4m3fn) for _ in range(2))
    ke, ve = (torch.zeros((2, kv, P), dtype=torch.uint8, device=DEV) for _ in range(2))
    q = torch.empty((1, heads, hd), dtype=torch.bfloat16, device=DEV)
    i32 = dict(dtype=torch.int32, device=DEV)
    K.rope_kv_write_e4m3(x, 0, 2 * hd, 3 * hd, q, k, v, ke, ve, torch.tensor([17], **i32), torch.tensor([0], **i32), torch.tensor([[1, 0]], **i32), P, heads, kv,
                         hd, 0, None, True)
    assert torch.equal(q.view(-1), x[0, :2 * hd].to(torch.bfloat16))
    for c, e, y in ((k, ke, x[0, 2 * hd:3 * hd]), (v, ve, x[0, 3 * hd:])):
        got = c[0, 0, 1].to(F64) * 2.0 ** (int(e[0, 0, 1]) - 127)
        assert ((got - y.to(F64)).abs() <= 2.0 ** -4 * y.abs() + 2.0 ** -10 * y.abs().amax()).all()
