"""4-bit weights at the limits of a call."""
import pytest
import torch

from oracle import w4 as ow4
from tests.gpu_util import require_gpu
from tests.test_gpu_w4 import laid_out, mlk

pytestmark = pytest.mark.gpu


def test_largest_number_of_slots():
    """The most slots there are, over the most experts: every work item of a launch is used.  A token's result does not depend
    on its place, so a part of the tokens alone, in tiles of the same size, gives the same bits."""
    dev = require_gpu()
    E, topk, H, I = 1024, 8, 32, 32
    T = (65535 - 1024) * 128 // topk
    a = laid_out(ow4.random_weights(2 * I, H, 32, torch.bfloat16, 1, False, (E,)), dev)
    b = laid_out(ow4.random_weights(H, I, 32, torch.bfloat16, 2, True, (E,)), dev)
    g = torch.Generator(device=dev).manual_seed(3)
    x = torch.randn(T, H, generator=g, device=dev).to(torch.bfloat16)
    ids = torch.randint(0, E, (T, topk), generator=g, device=dev, dtype=torch.int32)
    p = torch.rand(T, topk, generator=g, device=dev).to(torch.bfloat16)
    call = lambda rows: mlk().fused_experts_compute_w4(a[0], a[1], b[0], b[1], x[rows].contiguous(), ids[rows].contiguous(),  # noqa: E731
                                                       p[rows].contiguous(), w2_zeros=b[2])
    got = call(slice(0, T))
    for first in (0, T // 2, T - 20000):
        rows = slice(first, first + 20000)
        assert torch.equal(got[rows], call(rows))
    one_more = torch.zeros(T + 1, H, dtype=torch.bfloat16, device=dev)
    with pytest.raises(RuntimeError, match="slots"):
        mlk().fused_experts_compute_w4(a[0], a[1], b[0], b[1], one_more, torch.zeros(T + 1, topk, dtype=torch.int32, device=dev),
                                       torch.zeros(T + 1, topk, dtype=torch.bfloat16, device=dev), w2_zeros=b[2])
    assert mlk().kernel_status() == 0
