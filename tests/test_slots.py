"""Slots of a state cache moved by a row map (bm_slots_reorder) and with the
decode rows (bm_decode_reorder, bm_decode_compact): exact copies."""
import ctypes

import numpy as np
import pytest

import synth

DEFAULT = 1


def region(t):
    """A [n_outer, slots, ...] tensor (or a view with row pitch) as a region."""
    e = t.element_size()
    row = int(np.prod(t.shape[2:])) * e
    return (t.data_ptr(), row, t.stride(1) * e, t.shape[0], t.stride(0) * e)


def maps(S, kind, rng):
    src = np.arange(S)
    if kind == "rotate":
        src = np.roll(src, 1)
    elif kind == "reverse":
        src = src[::-1].copy()
    elif kind == "random":
        src = rng.integers(0, S, S)
    elif kind == "permute":
        src = rng.permutation(S)
    elif kind == "fork":
        src[:] = S // 2
    elif kind == "outside":
        src = rng.integers(-3, S + 3, S)
    elif kind == "few":
        src[rng.integers(0, S)] = rng.integers(0, S)
    return src


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["identity", "rotate", "reverse", "random", "permute", "fork", "outside", "few"])
@pytest.mark.parametrize("S", [1, 2, 7, 33, 257, 1024, 1025])
def test_reorder(gpu_ctx, sampler_lib, kind, S):
    import torch
    rng = np.random.default_rng(S)
    src = maps(S, kind, rng)
    g = torch.Generator(device="cuda").manual_seed(S)
    i32 = lambda *s: torch.randint(-2**31, 2**31 - 1, s, generator=g, device="cuda", dtype=torch.int32)  # noqa: E731
    # 16-byte rows, 4-byte rows, scalars, rows longer than a piece, pitched rows
    arrays = [i32(2, S, 24), i32(3, S, 7), i32(1, S, 1), i32(2, S, 2100 if S < 300 else 60), i32(1, S, 40)[:, :, :36]]
    want = []
    ok = (src >= 0) & (src < S)
    at = torch.from_numpy(np.where(ok, src, np.arange(S))).cuda()
    for a in arrays:
        want.append(a[:, at].clone())
    pad = arrays[4]._base.clone() if arrays[4]._base is not None else None
    d = torch.from_numpy(src.astype(np.int32)).cuda()
    torch.cuda.synchronize()
    gpu_ctx.slots_reorder(sampler_lib.slot_regions([region(a) for a in arrays]), d.data_ptr(), S, DEFAULT)
    torch.cuda.synchronize()
    for a, w in zip(arrays, want):
        assert torch.equal(a, w)
    if pad is not None:  # behind the pitched rows nothing changed
        assert torch.equal(arrays[4]._base[:, :, 36:], pad[:, :, 36:])


@pytest.mark.gpu
def test_reorder_most_slots(gpu_ctx, sampler_lib):
    import torch
    S = 8192
    a = torch.randint(0, 1 << 30, (1, S, 44), device="cuda", dtype=torch.int32)
    src = torch.randperm(S, device="cuda").to(torch.int32)
    want = a[:, src.long()].clone()
    torch.cuda.synchronize()
    gpu_ctx.slots_reorder(sampler_lib.slot_regions([region(a)]), src.data_ptr(), S, DEFAULT)
    torch.cuda.synchronize()
    assert torch.equal(a, want)


@pytest.mark.gpu
def test_reorder_captured(gpu_ctx, sampler_lib):
    import torch
    a = torch.arange(5 * 40 * 16, device="cuda", dtype=torch.int32).view(5, 40, 16).clone()
    src = torch.arange(40, device="cuda", dtype=torch.int32)
    r = sampler_lib.slot_regions([region(a)])
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        gpu_ctx.slots_reorder(r, src.data_ptr(), 40, torch.cuda.current_stream().cuda_stream)
    for k in range(3):
        src.copy_(torch.randperm(40, device="cuda"))
        want = a[:, src.long()].clone()
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(a, want)


def _decode(gpu_ctx, bm, B, seed, plants):
    """A decode state some steps in, with rows stopped at `plants`."""
    import torch
    V = synth.VOCAB
    rng = np.random.default_rng(seed)
    dec = bm.Decode(gpu_ctx, B, max_tokens=0, stop_ids=[777])
    dec.reset([list(rng.integers(1, 700, rng.integers(0, 300))) for _ in range(B)])
    kn = bm.knobs_array(0.0, 1.0, 0.0, 1.0, 0)  # greedy
    kd = torch.from_numpy(kn.view(np.uint8).copy()).cuda()
    u = torch.zeros(B, device="cuda")

    def step(want, rows=B):
        z = torch.zeros(rows, V, device="cuda")
        z[torch.arange(rows), torch.as_tensor(want, device="cuda")] = 5.0
        out = torch.full((B,), -7, dtype=torch.int32, device="cuda")
        torch.cuda.synchronize()
        dec.step(z.data_ptr(), V, V, kd.data_ptr(), 0, u.data_ptr(), out.data_ptr(), DEFAULT)
        torch.cuda.synchronize()
        return out.cpu().numpy()

    for k in range(3):
        want = rng.integers(1, 700, B)
        for r, at in plants:
            if at == k:
                want[r] = 777
        step(want)
    return dec, step


def _pushed(dec, B):
    """n_pushed from the device view."""
    import torch
    torch.cuda.synchronize()

    class View:
        __cuda_array_interface__ = {"shape": (B,), "typestr": "<i4", "version": 3,
                                    "data": (dec.views()["n_pushed"], False)}
    return torch.as_tensor(View(), device="cuda").cpu().numpy()


@pytest.mark.gpu
def test_decode_reorder(gpu_ctx, sampler_lib):
    """Rows forked and permuted: loop state, model state and active count."""
    import torch
    B = 13
    dec, step = _decode(gpu_ctx, sampler_lib, B, 3, [(2, 0), (7, 1), (12, 2)])
    before, pushed = dec.read(), _pushed(dec, B)
    src = np.array([0, 4, 2, 3, 7, 4, 4, -1, 8, 2, 99, 12, 11], np.int32)
    at = np.where((src >= 0) & (src < B), src, np.arange(B))
    state = torch.randn(3, B, 20, device="cuda")
    want = state[:, torch.from_numpy(at).cuda()].clone()
    d = torch.from_numpy(src).cuda()
    torch.cuda.synchronize()
    dec.reorder(d.data_ptr(), sampler_lib.slot_regions([region(state)]), DEFAULT)
    torch.cuda.synchronize()
    after = dec.read()
    for k in before:
        assert np.array_equal(after[k], before[k][at]), k
    assert np.array_equal(_pushed(dec, B), pushed[at])
    assert torch.equal(state, want)
    assert dec.active(DEFAULT) == int((after["status"] == 0).sum())
    ids = step(np.full(B, 55))
    assert np.array_equal(ids, np.where(after["status"] == 0, 55, -1))
    dec.close()


@pytest.mark.gpu
@pytest.mark.parametrize("B", [1, 5, 31, 1030])
def test_decode_compact(gpu_ctx, sampler_lib, B):
    import torch
    rng = np.random.default_rng(B)
    stopped = sorted(rng.permutation(B)[: B // 2])
    dec, step = _decode(gpu_ctx, sampler_lib, B, 4, [(r, int(rng.integers(0, 3))) for r in stopped])
    before = dec.read()
    assert np.array_equal(np.flatnonzero(before["status"]), stopped)
    live = np.setdiff1d(np.arange(B), stopped)
    order = np.concatenate([live, stopped]).astype(int)
    state = torch.randn(2, B, 12, device="cuda")
    want = state[:, torch.from_numpy(live).cuda()].clone()
    out = torch.empty(B, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    dec.compact(sampler_lib.slot_regions([region(state)]), out.data_ptr(), DEFAULT)
    torch.cuda.synchronize()
    after = dec.read()
    for k in before:
        assert np.array_equal(after[k], before[k][order]), k
    assert np.array_equal(out.cpu().numpy(), order)
    assert torch.equal(state[:, :len(live)], want)
    n = len(live)
    assert dec.active(DEFAULT) == n
    dec.set_rows(n)
    ids = step(np.full(n, 66), n)
    assert (ids[:n] == 66).all() and (ids[n:] == -7).all()
    final = dec.read()
    assert np.array_equal(final["n_generated"][n:], after["n_generated"][n:])
    dec.close()


def test_refusals(sampler_lib):
    bm = sampler_lib
    L = bm.lib()
    ctx = ctypes.create_string_buffer(1 << 16)
    q = 1 << 20

    def call(regions=((q, 64, 64, 2, 640),), src=q, S=10, ctx=ctx, n=None):
        a = bm.slot_regions(list(regions)) if regions is not None else None
        return L.bm_slots_reorder(ctx, a, len(regions or ()) if n is None else n, src, S, None)

    bad = [dict(ctx=None), dict(src=None), dict(src=q + 2), dict(S=-1), dict(S=8193), dict(n=9), dict(n=-1),
           dict(regions=None, n=1)]
    bad += [dict(regions=(r,)) for r in ((None, 64, 64, 2, 640), (q + 2, 64, 64, 2, 640), (q, 0, 64, 2, 640),
                                         (q, 66, 68, 2, 640), (q, 64, 60, 2, 640), (q, 64, 64, 0, 640),
                                         (q, 64, 66, 2, 640), (q, 64, 64, 2, 60), (q, 64, 64, 2, 641))]
    for b in bad:
        assert call(**b) in (-1, -4), b
    assert call(S=0) == 0 and call(regions=()) == 0
    for f, args in ((L.bm_decode_reorder, (None, q, None, 0, None)), (L.bm_decode_compact, (None, None, 0, None, None)),
                    (L.bm_decode_set_rows, (None, 1))):
        assert f(*args) == -1


@pytest.mark.gpu
def test_decode_compact_captured(gpu_ctx, sampler_lib):
    """A compaction in a graph, replayed after more rows have stopped."""
    import torch
    B = 40
    dec, step = _decode(gpu_ctx, sampler_lib, B, 6, [(3, 0), (20, 1)])
    state = torch.randn(3, B, 16, device="cuda")
    out = torch.empty(B, dtype=torch.int32, device="cuda")
    r = sampler_lib.slot_regions([region(state)])
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        dec.compact(r, out.data_ptr(), torch.cuda.current_stream().cuda_stream)
    for k in range(3):
        want = np.full(B, 50 + k)
        want[[5 + k, 11 * k]] = 777
        step(want)
        before, held = dec.read(), state.clone()
        live = np.flatnonzero(before["status"] == 0)
        order = np.concatenate([live, np.flatnonzero(before["status"])])
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        after = dec.read()
        for key in before:
            assert np.array_equal(after[key], before[key][order]), key
        assert np.array_equal(out.cpu().numpy(), order)
        assert torch.equal(state[:, :len(live)], held[:, torch.from_numpy(live).cuda()])
    dec.close()


def test_refuses_more_pieces_than_are_counted(sampler_lib):
    """Rows of a slot are cut into pieces of 16 bytes at least, whose number,
    with the rest of each row as one, stays in 31 bits (on the host; no slots,
    so nothing is launched)."""
    L = sampler_lib.lib()
    ctx = ctypes.create_string_buffer(1 << 16)
    q, most = 1 << 20, 2 ** 31 - 1

    def call(row, outer):
        return L.bm_slots_reorder(ctx, sampler_lib.slot_regions([(q, row, row, outer, row)]), 1, q, 0, None)

    assert call(16, most) == 0 and call(4, most) == 0 and call(32, most // 2) == 0
    assert call(20, most) == -1 and call(28, most // 2 + 1) == -1 and call(32, most // 2 + 1) == -1
