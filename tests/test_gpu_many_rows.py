"""More rows than one launch of the shape-agnostic GEMMs has workgroups for (a workgroup of 256 threads takes 32 rows; 2^32 threads)."""
import pytest
import torch

from avelang_amd import gemm_mxfp4_transposed_b
from tests import helpers as H

pytestmark = pytest.mark.gpu


def test_more_than_2_to_the_29_rows_of_one_output(gpu):
    m, n, k = (1 << 29) + 100, 1, 32
    g = torch.Generator(device=gpu).manual_seed(1)
    a = torch.randint(0, 256, (1 << 20, k // 2), dtype=torch.uint8, device=gpu, generator=g).repeat(m // (1 << 20) + 1, 1)[:m]
    a[-100:] = torch.randint(0, 256, (100, k // 2), dtype=torch.uint8, device=gpu, generator=g)
    a_s = torch.full((m, 1), 127, dtype=torch.uint8, device=gpu)
    b = torch.randint(0, 256, (n, k // 2), dtype=torch.uint8, device=gpu, generator=g)
    b_s = torch.full((n, 1), 126, dtype=torch.uint8, device=gpu)
    out = torch.full((m, n), float("nan"), dtype=torch.bfloat16, device=gpu)
    gemm_mxfp4_transposed_b(a, a_s, b, b_s, out)
    assert not out.isnan().any()
    assert (out[:1 << 29].view(-1, 1 << 20) == out[:1 << 20].view(-1)).all()
    rows = torch.cat([torch.arange(64, device=gpu), torch.arange(m - 130, m, device=gpu)])
    H.assert_mx_close(H.bits(out[rows]), a[rows].cpu().numpy(), a_s[rows].cpu().numpy(), b.cpu().numpy(), b_s.cpu().numpy())
