"""Failed calls of the layers' operators leave nothing behind: not in the
thread's CUDA error, not in the states."""
import ctypes

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


def test_workspace_growth(sampler_lib):
    """Twice the size, what is asked for, or the largest prompt's workspace
    (2^26 rows times heads), whichever ends the growing first; all buffers of
    one context come to less than three times the largest."""
    L = sampler_lib.lib()
    L.bm_detail_grown.restype = ctypes.c_size_t
    L.bm_detail_grown.argtypes = [ctypes.c_size_t, ctypes.c_size_t, ctypes.c_int]
    scan, fp8 = 0, 1
    most = max(-(-((1 << 26) // h) // lc) * h * (16 * lc + 4) for lc in (8, 16) for h in (1, 3, 7, 100, 4096, 32767, 65535, 65536))
    assert L.bm_detail_grown(0, 1000, scan) == 1024
    assert L.bm_detail_grown(1 << 20, (1 << 20) + 1, scan) == 2 << 20
    assert L.bm_detail_grown(1 << 20, 5 << 20, fp8) == 5 << 20
    assert most <= L.bm_detail_grown(int(1.09e9), int(1.1e9), scan) <= 1.13e9
    assert L.bm_detail_grown(1 << 40, (1 << 40) + 256, fp8) == 1 << 41
    for first in (256, 10 ** 6, most // 2 + 1):
        cap, kept = 0, 0
        need = first
        while need <= most:
            if need > cap:
                cap = L.bm_detail_grown(cap, need, scan)
                kept += cap
            need = cap + 256
        assert kept < 3 * 1.13e9 and cap >= most - 256


@pytest.mark.gpu
def test_workspace_grows_to_what_is_left(sampler_lib):
    """Where twice the old size cannot be had, what a call needs is enough."""
    import torch
    bm = sampler_lib
    ctx = bm.Context(0)
    d, n = 16384, 128
    x = torch.randn(20480, d, device="cuda")
    w = torch.randn(n, d, device="cuda").to(torch.float8_e4m3fn)
    ws = torch.ones(1, d // 128, device="cuda")
    out = torch.empty(20480, n, device="cuda")

    def call(rows):
        torch.cuda.synchronize()
        ctx.fp8_logits(x.data_ptr(), rows, d, None, w.data_ptr(), ws.data_ptr(), n, out.data_ptr(), n, DEFAULT)
        torch.cuda.synchronize()

    call(16384)  # 256 MB and the scales
    small = out[:16384].clone()
    torch.cuda.empty_cache()
    free = torch.cuda.mem_get_info()[0]
    rest = torch.empty(free - (450 << 20), dtype=torch.uint8, device="cuda")
    try:
        assert torch.cuda.mem_get_info()[0] < 520 << 20  # no room for twice 264 MB
        call(20480)
    finally:
        del rest
        torch.cuda.empty_cache()
    assert torch.equal(out[:16384], small)
    ctx.check()
    ctx.close()
