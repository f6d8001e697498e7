"""CPU tests of the choice that the experts' products are given: it is an operand, not a buffer that a call may make."""
import pytest
import torch

import gq


@pytest.mark.parametrize("ids,weights", [(None, None), (torch.zeros(4, 2, dtype=torch.int32), None), (None, torch.zeros(4, 2)),
                                         (torch.zeros(8, dtype=torch.int32), torch.zeros(4, 2))])
def test_a_choice_is_required(ids, weights):
    x, w = torch.zeros(4, 256, dtype=torch.bfloat16), torch.zeros(gq.packed_size(gq.FMT_Q4_0, 8 * 64, 256), dtype=torch.uint8)
    d = torch.zeros(gq.packed_size(gq.FMT_Q4_0, 8 * 256, 64), dtype=torch.uint8)
    with pytest.raises(gq.GQError, match="ids and weights"):
        gq.moe_ffn(gq.FMT_Q4_0, w, w, gq.FMT_Q4_0, d, x, ids, weights, 64, 256, 8)


@pytest.mark.gpu
def test_a_choice_is_an_operand(dev):
    """On the device: none, another shape or type, host memory."""
    x, w = torch.zeros(4, 256, dtype=torch.bfloat16, device=dev), torch.zeros(gq.packed_size(gq.FMT_Q4_0, 8 * 64, 256), dtype=torch.uint8, device=dev)
    d = torch.zeros(gq.packed_size(gq.FMT_Q4_0, 8 * 256, 64), dtype=torch.uint8, device=dev)
    ids, weights = torch.zeros(4, 2, dtype=torch.int32, device=dev), torch.zeros(4, 2, device=dev)

    def call(ids, weights):
        return gq.moe_ffn(gq.FMT_Q4_0, w, w, gq.FMT_Q4_0, d, x, ids, weights, 64, 256, 8)

    for bad in ((None, weights), (ids, None), (ids.long(), weights), (ids, weights.half()), (ids[:3], weights), (ids, weights[:, :1]),
                (ids.cpu(), weights), (ids, weights.cpu()), (ids, weights.t().contiguous().t())):
        with pytest.raises(gq.GQError):
            call(*bad)
    assert bool((call(ids, weights) == 0).all())
