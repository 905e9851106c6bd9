"""Failed calls of the layers' operators leave nothing behind: not in the
thread's CUDA error, not in the states."""
import numpy as np
import pytest

from test_ssm import DEFAULT, Problem


@pytest.mark.gpu
def test_calls_after_a_failed_workspace(sampler_lib):
    """A workspace larger than the device (17 TB) is refused; the calls behind
    it launch, report that, and take their token or move once."""
    import torch
    bm = sampler_lib
    ctx = bm.Context(0)
    w = torch.zeros(1 << 14, device="cuda")

    def too_large():
        with pytest.raises(bm.BmError) as e:
            ctx.fp8_logits(w.data_ptr(), 1 << 30, 16384, None, w.data_ptr(), w.data_ptr(), 8, w.data_ptr(), 8, DEFAULT)
        assert e.value.code == -3

    p = Problem(1, "f32", 2, 32, 3, 3)
    torch.cuda.synchronize()
    too_large()
    p.step(bm, ctx)
    p.check(list(range(4)), fresh=[0] * 3)

    state = torch.randn(4, 5, 8, device="cuda")
    want = state[:, [4, 0, 1, 2, 3]].clone()
    src = torch.tensor([4, 0, 1, 2, 3], dtype=torch.int32, device="cuda")
    regions = bm.slot_regions([(state.data_ptr(), 32, 32, 4, 5 * 32)])
    torch.cuda.synchronize()
    too_large()
    ctx.slots_reorder(regions, src.data_ptr(), 5, DEFAULT)
    torch.cuda.synchronize()
    assert torch.equal(state, want)

    dec = bm.Decode(ctx, 5, 3)
    dec.reset([[1, 2], [3], [4, 5, 6], [7], [8, 9]])
    too_large()
    dec.reorder(src.data_ptr(), regions, DEFAULT)
    too_large()
    dec.compact(regions, None, DEFAULT)
    torch.cuda.synchronize()
    assert torch.equal(state, want[:, [4, 0, 1, 2, 3]])
    assert np.array_equal(dec.read()["current"], [9, 2, 3, 6, 7])

    x = torch.randn(7, 128, device="cuda")
    q, scale = torch.empty(7, 128, dtype=torch.uint8, device="cuda"), torch.empty(1, 8, device="cuda")
    torch.cuda.synchronize()
    too_large()
    ctx.fp8_quantize(x.data_ptr(), "f32", 7, 128, 128, None, q.data_ptr(), scale.data_ptr(), 8, DEFAULT)
    p = Problem(2, "f32", 2, 32, 1500, 1)
    torch.cuda.synchronize()
    too_large()
    p.prefill(bm, ctx, [0, 1500])
    p.check([0, 1500])
    ctx.check()
    dec.close()
    ctx.close()
