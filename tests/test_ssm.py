"""The state space mixer (bm_ssm_prefill, bm_ssm_step) against its definition
in 64 bits (tests/ssm_ref.py, which derives the bounds)."""
import ctypes

import numpy as np
import pytest

import ssm_ref

DEFAULT = 1  # cudaStreamLegacy: the stream torch works on in these tests


class Problem:
    """Random inputs on the host (rounded to the type) and the device."""

    def __init__(self, seed, type_, H, P, rows, n_slots, gate=True, pad=0):
        import torch
        self.torch = torch
        rng = np.random.default_rng(seed)
        self.type, self.H, self.P, self.C, self.rows, self.n_slots = type_, H, P, H * P, rows, n_slots
        self.t = torch.float32 if type_ == "f32" else torch.bfloat16
        self.gate = gate
        self.ld = 2 * self.C + 3 * H + pad
        self.w = ssm_ref.weights(rng, H, P)
        self.proj = torch.from_numpy(rng.standard_normal((max(rows, 1), self.ld)).astype(np.float32)).to(self.t)
        self.conv = torch.from_numpy(rng.standard_normal((n_slots, 3, self.C)).astype(np.float32)).to(self.t)
        self.h = torch.from_numpy(rng.standard_normal((n_slots, self.C)).astype(np.float32))
        self.dev = {k: torch.from_numpy(v).cuda() for k, v in self.w.items()}
        self.dproj, self.dconv, self.dh = self.proj.cuda(), self.conv.cuda(), self.h.cuda()
        self.y = torch.full((max(rows, 1), self.C), 7.0, dtype=self.t, device="cuda")

    def layer(self, bm):
        return bm.SsmLayer(self.H, self.P, self.n_slots, self.type,
                           **{k: v.data_ptr() for k, v in self.dev.items()},
                           conv_state=self.dconv.data_ptr(), h_state=self.dh.data_ptr())

    def ptrs(self):
        e, at, C, H = self.proj.element_size(), self.dproj.data_ptr(), self.C, self.H
        z = at if self.gate else None
        return at + C * e, z, at + 2 * C * e, at + (2 * C + H) * e, at + (2 * C + 2 * H) * e

    def prefill(self, bm, ctx, off, slots=None, fresh=None, rows=None, stream=DEFAULT):
        i = lambda a, t: None if a is None else self.torch.tensor(a, dtype=t, device="cuda")  # noqa: E731
        self.keep = [i(off, self.torch.int64), i(slots, self.torch.int32), i(fresh, self.torch.int32)]
        o, s, f = self.keep
        ctx.ssm_prefill(self.layer(bm), *self.ptrs(), self.ld, self.rows if rows is None else rows,
                        o.data_ptr(), len(off) - 1, None if s is None else s.data_ptr(),
                        None if f is None else f.data_ptr(), self.y.data_ptr(), self.C, stream)

    def step(self, bm, ctx, slots=None, stream=DEFAULT):
        self.keep = self.torch.tensor(slots, dtype=self.torch.int32, device="cuda") if slots is not None else None
        ctx.ssm_step(self.layer(bm), *self.ptrs(), self.ld, self.rows,
                     None if slots is None else self.keep.data_ptr(), self.y.data_ptr(), self.C, stream)

    def check(self, off, slots=None, fresh=None):
        """Everything that a call may write, and that nothing else changed."""
        self.torch.cuda.synchronize()
        f = self.proj.double().numpy()
        C, H = self.C, self.H
        z, x = f[:, :C], f[:, C:2 * C]
        b, c, dt = (f[:, 2 * C + k * H:2 * C + (k + 1) * H] for k in range(3))
        w = {k: v.astype(np.float64) for k, v in self.w.items()}
        conv, h = self.conv.double().numpy(), self.h.double().numpy()
        eh, ey = np.zeros_like(h), np.zeros((f.shape[0], C))
        y = np.full((f.shape[0], C), 7.0)
        n = len(off) - 1
        for i in range(n):
            s = i if slots is None else slots[i]
            if not 0 <= s < self.n_slots:
                continue
            r = slice(max(0, off[i]), min(self.rows, off[i + 1]))
            new = fresh is None or bool(fresh[i])
            y[r], ey[r], conv[s], h[s], eh[s] = ssm_ref.run(
                x[r], z[r] if self.gate else None, b[r], c[r], dt[r], w, H, self.P, conv[s], h[s], new)
        got_y = self.y.double().cpu().numpy()
        half = 2.0 ** -8 if self.type == "bf16" else ssm_ref.U
        bad = np.abs(got_y - y) > ey * 1.01 + half * np.abs(y) + 1e-30
        assert not bad.any(), (np.argwhere(bad)[:5], got_y[bad][:5], y[bad][:5], ey[bad][:5])
        got_h = self.dh.double().cpu().numpy()
        bad = np.abs(got_h - h) > eh * 1.01 + 1e-30
        assert not bad.any(), (np.argwhere(bad)[:5], got_h[bad][:5], h[bad][:5], eh[bad][:5])
        assert np.array_equal(self.dconv.double().cpu().numpy(), conv)


def offsets(lengths, first=0):
    return [first] + list(np.cumsum(lengths) + first)


LENGTHS = [[1], [2], [3], [4], [5], [31], [32], [33], [63], [64], [65], [300], [1, 1, 1], [0, 5, 0, 0, 3],
           [2, 1, 3, 1, 40, 1], [30, 2, 1, 33, 64, 0, 7], [0], [1] * 70, [129, 127, 128, 200]]
SHAPES = [(1, 1), (3, 5), (2, 16), (5, 24), (4, 64), (3, 130), (9, 40), (33, 4)]


@pytest.mark.gpu
@pytest.mark.parametrize("type_", ["f32", "bf16"])
@pytest.mark.parametrize("k", range(len(LENGTHS)))
def test_prefill(gpu_ctx, sampler_lib, type_, k):
    lengths = LENGTHS[k]
    H, P = SHAPES[k % len(SHAPES)]
    n = len(lengths)
    off = offsets(lengths)
    rng = np.random.default_rng(k)
    p = Problem(k, type_, H, P, off[-1], n + 2, gate=k % 3 != 1, pad=k % 4)
    slots = list(rng.permutation(n + 2)[:n])
    fresh = list((rng.random(n) < 0.5).astype(int))
    p.prefill(sampler_lib, gpu_ctx, off, slots, fresh)
    p.check(off, slots, fresh)
    gpu_ctx.check()


@pytest.mark.gpu
@pytest.mark.parametrize("type_", ["f32", "bf16"])
@pytest.mark.parametrize("shape", SHAPES)
def test_prefill_shapes(gpu_ctx, sampler_lib, type_, shape):
    off = offsets([70, 33])
    p = Problem(5, type_, *shape, off[-1], 2)
    p.prefill(sampler_lib, gpu_ctx, off)
    p.check(off)


@pytest.mark.gpu
@pytest.mark.parametrize("type_", ["f32", "bf16"])
def test_prefill_rows_of_no_sequence(gpu_ctx, sampler_lib, type_):
    """Rows before the first and behind the last sequence and those of
    sequences without a valid slot are left as they were."""
    off = offsets([10, 40, 37, 3], first=6)
    p = Problem(6, type_, 3, 24, off[-1] + 50, 5)
    slots, fresh = [4, -1, 0, 5], [0, 0, 1, 0]
    p.prefill(sampler_lib, gpu_ctx, off, slots, fresh)
    p.check(off, slots, fresh)


@pytest.mark.gpu
def test_prefill_offsets_beyond_the_rows(gpu_ctx, sampler_lib):
    """Offsets behind the last row (a stale count) reach no memory there: the
    sequences end at the last row."""
    p = Problem(8, "f32", 2, 40, 50, 3)
    p.prefill(sampler_lib, gpu_ctx, [0, 20, 90, 200])
    p.torch.cuda.synchronize()
    q = Problem(8, "f32", 2, 40, 50, 3)
    q.prefill(sampler_lib, gpu_ctx, [0, 20, 50, 50])
    p.torch.cuda.synchronize()
    assert p.torch.equal(p.y, q.y)


@pytest.mark.gpu
@pytest.mark.parametrize("type_", ["f32", "bf16"])
def test_prefill_in_parts_equals_whole(gpu_ctx, sampler_lib, type_):
    """A prompt in three calls, each continuing the slot, against one call."""
    T, cuts = 333, [0, 2, 131, 333]
    p = Problem(9, type_, 4, 48, T, 1)
    p.prefill(sampler_lib, gpu_ctx, [0, T])
    p.check([0, T])
    q = Problem(9, type_, 4, 48, T, 1)
    for a, b in zip(cuts, cuts[1:]):
        # the sequence's rows within the same arrays: rows of no sequence are left
        q.prefill(sampler_lib, gpu_ctx, [a, b], [0], [int(a == 0)])
    q.check([0, T])


@pytest.mark.gpu
@pytest.mark.parametrize("type_", ["f32", "bf16"])
def test_prefill_long_many_tiles(gpu_ctx, sampler_lib, type_):
    """Thousands of rows: states carried over many tiles, sequence ends
    anywhere among them, twice in a row on the same workspace."""
    off = offsets([2000, 1, 777, 1500])
    p = Problem(10, type_, 2, 64, off[-1], 4)
    p.prefill(sampler_lib, gpu_ctx, off)
    p.prefill(sampler_lib, gpu_ctx, off)
    p.check(off)
    gpu_ctx.check()


@pytest.mark.gpu
@pytest.mark.parametrize("type_", ["f32", "bf16"])
@pytest.mark.parametrize("H,P,rows,pad", [(16, 128, 600, 0), (9, 24, 2300, 0), (4, 64, 2300, 2), (3, 16, 2200, 4), (16, 64, 2100, 6),
                                          (5, 7, 2100, 0), (64, 16, 300, 0), (2, 80, 4200, 8)])
def test_prefill_tall(gpu_ctx, sampler_lib, type_, H, P, rows, pad):
    """The ways of the taller prompts: clusters of two to eight, head scalars
    from a launch of their own, copies of 16 bytes and of single words, heads
    across the edges of a CTA's channels."""
    off = offsets([rows // 3, 2, rows - rows // 3 - 2])
    p = Problem(rows + P, type_, H, P, rows, 4, pad=pad)
    p.prefill(sampler_lib, gpu_ctx, off, [2, 0, 3], [0, 0, 1])
    p.check(off, [2, 0, 3], [0, 0, 1])


@pytest.mark.gpu
@pytest.mark.parametrize("type_", ["f32", "bf16"])
@pytest.mark.parametrize("gate", [True, False])
@pytest.mark.parametrize("seed,H,P,most", [(1, 2, 32, 20), (2, 3, 32, 60), (3, 2, 48, 300), (4, 20, 128, 900)])
def test_prefill_ragged_tall(gpu_ctx, sampler_lib, type_, gate, seed, H, P, most):
    """Boundaries at every place of a part and of a tile, states taken up and
    started, rows of no sequence before the first and behind the last."""
    rng = np.random.default_rng(seed)
    lengths = []
    while sum(lengths) < 2600:
        lengths.append(int(rng.integers(0, most)))
    n = len(lengths)
    off = offsets(lengths, first=7)
    p = Problem(seed, type_, H, P, off[-1] + 30, n + 2, gate=gate)
    slots, fresh = list(rng.permutation(n + 2)[:n]), list((rng.random(n) < 0.5).astype(int))
    p.prefill(sampler_lib, gpu_ctx, off, slots, fresh)
    p.check(off, slots, fresh)


@pytest.mark.gpu
@pytest.mark.parametrize("type_", ["f32", "bf16"])
def test_prefill_thousands_of_sequences(gpu_ctx, sampler_lib, type_):
    """More sequences than a CTA keeps offsets of; many without tokens."""
    rng = np.random.default_rng(2)
    lengths = list(rng.integers(0, 4, 1500))
    off = offsets(lengths)
    p = Problem(17, type_, 2, 16, off[-1], 1600)
    slots = list(rng.permutation(1600)[:1500])
    fresh = list((rng.random(1500) < 0.5).astype(int))
    p.prefill(sampler_lib, gpu_ctx, off, slots, fresh)
    p.check(off, slots, fresh)


@pytest.mark.gpu
def test_prefill_is_reproducible(gpu_ctx, sampler_lib):
    """The order in which tiles finish does not show in the results."""
    off = offsets([3000])
    out = []
    for _ in range(4):
        p = Problem(11, "f32", 4, 128, off[-1], 1)
        p.prefill(sampler_lib, gpu_ctx, off)
        p.torch.cuda.synchronize()
        out.append((p.y.clone(), p.dh.clone()))
    for y, h in out[1:]:
        assert p.torch.equal(y, out[0][0]) and p.torch.equal(h, out[0][1])


@pytest.mark.gpu
def test_prefill_extreme_steps(gpu_ctx, sampler_lib):
    """Steps so large that a state is forgotten at once (the decay underflows)
    and so small that it never is."""
    off = offsets([200])
    for value in (90.0, -90.0):
        p = Problem(12, "f32", 2, 32, 200, 1)
        C, H = p.C, p.H
        p.proj[:, 2 * C + 2 * H:2 * C + 3 * H] = value
        p.dproj = p.proj.cuda()
        p.prefill(sampler_lib, gpu_ctx, off)
        p.check(off)


@pytest.mark.gpu
def test_prefill_nan_and_infinity_stay_in_their_sequence(gpu_ctx, sampler_lib):
    off = offsets([40, 41, 50])
    p = Problem(13, "f32", 2, 32, off[-1], 3)
    q = Problem(13, "f32", 2, 32, off[-1], 3)
    p.dproj[45, p.C:2 * p.C] = float("nan")
    p.dproj[60, p.C:2 * p.C] = float("inf")
    p.prefill(sampler_lib, gpu_ctx, off)
    q.prefill(sampler_lib, gpu_ctx, off)
    p.torch.cuda.synchronize()
    for a, b in ((0, 45), (81, 131)):
        assert p.torch.equal(p.y[a:b], q.y[a:b])
    assert p.y[45:81].isnan().any(1).all()
    assert p.torch.equal(p.dh[[0, 2]], q.dh[[0, 2]]) and p.dh[1].isnan().all()


@pytest.mark.gpu
@pytest.mark.parametrize("type_", ["f32", "bf16"])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("rows", [1, 2, 37, 300])
def test_step(gpu_ctx, sampler_lib, type_, shape, rows):
    rng = np.random.default_rng(rows)
    p = Problem(rows, type_, *shape, rows, rows + 4, gate=rows != 2, pad=rows % 4)
    slots = list(rng.permutation(rows + 4)[:rows])
    if rows > 5:
        slots[3], slots[5] = -1, rows + 4  # skipped
    p.step(sampler_lib, gpu_ctx, slots)
    p.check(list(range(rows + 1)), slots, [0] * rows)
    gpu_ctx.check()


@pytest.mark.gpu
@pytest.mark.parametrize("type_", ["f32", "bf16"])
def test_steps_continue_a_prompt(gpu_ctx, sampler_lib, type_):
    """A prompt then single tokens give what the whole sequence gives."""
    T, n = 75, 11
    p = Problem(14, type_, 3, 32, T, 1)
    p.prefill(sampler_lib, gpu_ctx, [0, n])
    x, z, b, c, dt = p.ptrs()
    e = p.proj.element_size()
    for t in range(n, T):
        o = t * p.ld * e
        gpu_ctx.ssm_step(p.layer(sampler_lib), x + o, z + o, b + o, c + o, dt + o, p.ld, 1, None,
                         p.y.data_ptr() + t * p.C * e, p.C, DEFAULT)
    p.check([0, T])


@pytest.mark.gpu
def test_captured_and_replayed(gpu_ctx, sampler_lib):
    """Prefill and steps in a CUDA graph on a stream of their own, replayed on
    changed inputs, with eager calls of other sizes in between."""
    import torch
    off, T = [0, 500, 1200], 1200
    p = Problem(15, "f32", 4, 64, T, 2)
    o = torch.tensor(off, device="cuda")
    layer = p.layer(sampler_lib)

    def calls(stream):
        gpu_ctx.ssm_prefill(layer, *p.ptrs(), p.ld, T, o.data_ptr(), 2, None, None, p.y.data_ptr(), p.C, stream)
        gpu_ctx.ssm_step(layer, *p.ptrs(), p.ld, 2, None, p.y.data_ptr(), p.C, stream)

    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    calls(s.cuda_stream)  # the first call of a size is not captured
    s.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        calls(torch.cuda.current_stream().cuda_stream)
    big = Problem(16, "f32", 4, 64, 9000, 1)  # grows the workspace
    for k in range(3):
        new = Problem(20 + k, "f32", 4, 64, T, 2)
        p.dproj.copy_(new.dproj)
        torch.cuda.synchronize()
        big.prefill(sampler_lib, gpu_ctx, [0, 9000])
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        y, h = p.y.clone(), p.dh.clone()
        p.y.fill_(7.0)
        torch.cuda.synchronize()
        calls(DEFAULT)
        torch.cuda.synchronize()
        # the replay continued nothing: every sequence started from zero, then took one token
        assert torch.equal(y, p.y) and torch.equal(h, p.dh)
    gpu_ctx.check()


@pytest.mark.gpu
def test_prefill_far_from_zero(gpu_ctx, sampler_lib):
    """Sigmoids at their ends: inputs and gates of hundreds, next to small ones
    in the same pair of channels; compared to the largest of each row."""
    import torch
    p = Problem(36, "f32", 2, 32, 200, 1)
    g = torch.Generator().manual_seed(3)
    scale = torch.exp2(torch.randint(-8, 9, (200, 4 * 32), generator=g).float())
    p.proj[:, :2 * p.C] *= scale
    p.dproj.copy_(p.proj)
    torch.cuda.synchronize()
    p.prefill(sampler_lib, gpu_ctx, [0, 200])
    torch.cuda.synchronize()
    f = p.proj.double().numpy()
    C, H = p.C, p.H
    w = {k: v.astype(np.float64) for k, v in p.w.items()}
    y, ey, _, h, _ = ssm_ref.run(f[:, C:2 * C], f[:, :C], *(f[:, 2 * C + k * H:2 * C + (k + 1) * H] for k in range(3)), w, H,
                                 p.P, np.zeros((3, C)), np.zeros(C), True)
    got = p.y.double().cpu().numpy()
    top = np.abs(y).max(1, keepdims=True)
    assert np.isfinite(got).all()
    assert (np.abs(got - y) <= 2 * ey + ssm_ref.U * np.abs(y) + 2.0 ** -40 * top).all()


def refused(call, args, **changes):
    a = dict(args)
    a.update(changes)
    return call(*a.values())


def test_refusals(sampler_lib):
    """On the host, before anything is launched: each bad argument alone (the
    context stands for a real one; a refused call never reads it)."""
    bm = sampler_lib
    L = bm.lib()
    ctx = ctypes.create_string_buffer(1 << 16)
    q = 1 << 20  # an aligned address that is never read

    def layer(**kw):
        a = dict(n_heads=4, head_dim=8, n_slots=3, type="f32")
        w = dict(conv_w=q, conv_b=q, dt_bias=q, a_log=q, d=q, conv_state=q, h_state=q)
        for k, v in kw.items():
            (a if k in a else w)[k] = v
        t = a.pop("type")
        s = bm.SsmLayer(a["n_heads"], a["head_dim"], a["n_slots"], t if isinstance(t, str) else "f32", **w)
        if not isinstance(t, str):
            s.struct.type = t
        return s.ref

    base = dict(ctx=ctx, layer=layer(), x=q, z=q, b=q, c=q, dt=q, ld=80, rows=5, off=q, n_seq=2, slots=q,
                fresh=q, y=q, ldy=32, stream=None)
    step = {k: v for k, v in base.items() if k not in ("off", "n_seq", "fresh")}
    step["rows"] = 3
    both = [dict(ctx=None), dict(layer=None), dict(layer=layer(n_heads=0)), dict(layer=layer(head_dim=0)),
            dict(layer=layer(n_slots=0)), dict(layer=layer(type=2)), dict(layer=layer(n_heads=1 << 18)),
            dict(layer=layer(conv_w=None)), dict(layer=layer(h_state=None)), dict(layer=layer(conv_state=None)),
            dict(layer=layer(conv_w=q + 4)), dict(layer=layer(h_state=q + 2)), dict(layer=layer(a_log=q + 1)),
            dict(x=None), dict(b=None), dict(c=None), dict(dt=None), dict(y=None), dict(x=q + 2), dict(y=q + 1),
            dict(z=q + 1), dict(ld=31), dict(ldy=31), dict(rows=-1)]
    for ch in both:
        assert refused(L.bm_ssm_prefill, base, **ch) in (-1, -4), ch
        assert refused(L.bm_ssm_step, step, **ch) in (-1, -4), ch
    for ch in (dict(off=None), dict(off=q + 4), dict(n_seq=-1), dict(n_seq=4)):
        assert refused(L.bm_ssm_prefill, base, **ch) in (-1, -4), ch
    assert refused(L.bm_ssm_step, step, rows=4) == -1  # more rows than slots
    assert refused(L.bm_ssm_step, step, rows=0) == 0
    assert refused(L.bm_ssm_prefill, base, n_seq=0) == 0
    with pytest.raises(ValueError):
        bm.SsmLayer(1, 1, 1, "f16", conv_w=q, conv_b=q, dt_bias=q, a_log=q, d=q, conv_state=q, h_state=q)


@pytest.mark.gpu
def test_captured_with_the_workspace(gpu_ctx, sampler_lib):
    """A prompt long enough for the workspace, captured, then replayed after a
    longer one has grown it: the graph still has its own."""
    import torch
    T = 2500
    p = Problem(31, "bf16", 3, 32, T, 2)
    o = torch.tensor([0, 700, T], device="cuda")
    layer = p.layer(sampler_lib)

    def call(stream):
        gpu_ctx.ssm_prefill(layer, *p.ptrs(), p.ld, T, o.data_ptr(), 2, None, None, p.y.data_ptr(), p.C, stream)

    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    call(s.cuda_stream)
    s.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        call(torch.cuda.current_stream().cuda_stream)
    big = Problem(32, "bf16", 40, 16, 6000, 1)
    big.prefill(sampler_lib, gpu_ctx, [0, 6000])
    big.check([0, 6000])
    p.y.fill_(7.0)
    p.dh.copy_(p.h)
    p.dconv.copy_(p.conv)
    torch.cuda.synchronize()
    g.replay()
    p.check([0, 700, T])


@pytest.mark.gpu
def test_two_contexts_at_once(gpu_ctx, sampler_lib):
    """Prompts that use the workspace, on two contexts and two streams with
    nothing between them."""
    import torch
    other = sampler_lib.Context(0)
    a, b = Problem(33, "f32", 4, 32, 4000, 1), Problem(34, "f32", 4, 32, 4000, 1)
    sa, sb = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    o = torch.tensor([0, 4000], device="cuda")
    torch.cuda.synchronize()
    for _ in range(3):
        for ctx, p, s in ((gpu_ctx, a, sa), (other, b, sb)):
            ctx.ssm_prefill(p.layer(sampler_lib), *p.ptrs(), p.ld, 4000, o.data_ptr(), 1, None, None, p.y.data_ptr(),
                            p.C, s.cuda_stream)
    a.check([0, 4000])
    b.check([0, 4000])
    other.close()


@pytest.mark.gpu
def test_prefill_of_nothing(gpu_ctx, sampler_lib):
    """No rows, no inputs: fresh slots are zeroed, the others stay."""
    import torch
    p = Problem(35, "f32", 2, 24, 0, 5)
    slots, fresh = [3, 1, 9, 0], [1, 0, 1, 1]
    i = [torch.tensor(v, dtype=torch.int32, device="cuda") for v in (slots, fresh)]
    o = torch.zeros(5, dtype=torch.int64, device="cuda")
    torch.cuda.synchronize()
    gpu_ctx.ssm_prefill(p.layer(sampler_lib), None, None, None, None, None, 0, 0, o.data_ptr(), 4, i[0].data_ptr(),
                        i[1].data_ptr(), None, 0, DEFAULT)
    p.check([0] * 5, slots, fresh)


def test_refuses_lists_off_their_alignment(sampler_lib):
    L = sampler_lib.lib()
    ctx = ctypes.create_string_buffer(1 << 16)
    q = 1 << 20
    layer = sampler_lib.SsmLayer(4, 8, 3, "f32", conv_w=q, conv_b=q, dt_bias=q, a_log=q, d=q, conv_state=q, h_state=q).ref
    for slots, fresh in ((q + 2, q), (q, q + 2), (q + 1, None)):
        assert L.bm_ssm_prefill(ctx, layer, q, q, q, q, q, 80, 5, q, 2, slots, fresh, q, 32, None) == -1
    assert L.bm_ssm_step(ctx, layer, q, q, q, q, q, 80, 3, q + 2, q, 32, None) == -1


def strongly_negative(p, seed, mid):
    """Some of a problem's gates and inputs replaced by -1e4 to -3e38 (as many
    gates by -44 to -85 with `mid`), the convolution reduced to the newest
    input; returns a mask over the projection's columns of the former."""
    import torch
    g = torch.Generator().manual_seed(seed)
    n = 2 * p.C
    far = torch.tensor([-1e4, -1e12, -1e19, -1e20, -1e30, -3e38])
    pick = torch.rand(p.proj.shape[0], n, generator=g)
    values = far[torch.randint(0, len(far), pick.shape, generator=g)].to(p.t)
    hit = torch.zeros(p.proj.shape, dtype=torch.bool)
    hit[:, :n] = pick < 0.3
    p.proj[:, :n] = torch.where(hit[:, :n], values, p.proj[:, :n])
    if mid:
        between = (-44 - 41 * torch.rand(pick[:, :p.C].shape, generator=g)).to(p.t)
        p.proj[:, :p.C] = torch.where(pick[:, :p.C] > 0.7, between, p.proj[:, :p.C])
    p.dproj.copy_(p.proj)
    p.conv.zero_()
    p.dconv.zero_()
    p.w["conv_b"][:] = 0
    p.w["conv_w"][:] = [0, 0, 0, 1]
    p.dev["conv_b"].zero_()
    p.dev["conv_w"].copy_(torch.from_numpy(p.w["conv_w"]))
    torch.cuda.synchronize()
    return hit


@pytest.mark.gpu
@pytest.mark.parametrize("type_", ["f32", "bf16"])
@pytest.mark.parametrize("P", [32, 15, 4])
@pytest.mark.parametrize("rows", [40, 300, 2500])
def test_sigmoids_of_strongly_negative_values(gpu_ctx, sampler_lib, type_, P, rows):
    """silu is 0 far below 0 whatever the magnitude, next to ordinary channels,
    and as exact between: what a prompt gives with such inputs and gates is what
    the formula gives with zeros in their place (silu(0) = 0 too)."""
    import torch
    p = Problem(40, type_, 4, P, rows, 1)
    hit = strongly_negative(p, rows, True)
    p.prefill(sampler_lib, gpu_ctx, [0, rows])
    torch.cuda.synchronize()
    last = p.proj[-3:, p.C:2 * p.C].clone()
    assert torch.equal(p.dconv[0].cpu(), last)
    p.proj[hit] = 0.0
    p.dconv[0] = p.proj[-3:, p.C:2 * p.C].cuda()
    p.check([0, rows])
    gpu_ctx.check()


@pytest.mark.gpu
@pytest.mark.parametrize("type_", ["f32", "bf16"])
@pytest.mark.parametrize("P", [32, 15])
def test_step_with_strongly_negative_values(gpu_ctx, sampler_lib, type_, P):
    import torch
    p = Problem(41, type_, 4, P, 20, 20)
    hit = strongly_negative(p, 5, True)
    p.step(sampler_lib, gpu_ctx)
    torch.cuda.synchronize()
    assert torch.equal(p.dconv[:, 2].cpu(), p.proj[:, p.C:2 * p.C])
    p.proj[hit] = 0.0
    # One step from a state s: a s is off by err(a) |s| where ssm_ref.run, which
    # bounds sums of many terms, has err(a) (a |s| + |g u|).  So its bound is
    # widened by err(a) |s|, and the output's by that times |C silu(z)|, with
    # err(a) as derived there: (13 |arg| + 4) u + 8 u d rate + u |v| rate
    # relative for a = exp(-arg), arg = rate d, d = softplus(v).
    f = p.proj.double().numpy()
    C, H, u = p.C, p.H, ssm_ref.U
    w = {k: v.astype(np.float64) for k, v in p.w.items()}
    half = 2.0 ** -8 if type_ == "bf16" else u
    for r in range(20):
        z, x = f[r:r + 1, :C], f[r:r + 1, C:2 * C]
        b, c, dt = (f[r:r + 1, 2 * C + k * H:2 * C + (k + 1) * H] for k in range(3))
        h0 = p.h[r].double().numpy()
        y, ey, _, h, eh = ssm_ref.run(x, z, b, c, dt, w, H, P, np.zeros((3, C)), h0, False)
        v, rate = dt[0] + w["dt_bias"], np.exp(w["a_log"])
        arg = rate * np.logaddexp(v, 0.0)
        ea = ((13 * arg + 4) + 8 * arg + rate * np.abs(v)) * u * np.exp(-arg)
        more = ea.repeat(P) * np.abs(h0)
        got_h, got_y = p.dh[r].double().cpu().numpy(), p.y[r].double().cpu().numpy()
        assert (np.abs(got_h - h) <= (eh + more) * 1.01 + 1e-30).all()
        gate = np.abs(c[0].repeat(P) * z[0] / (1.0 + np.exp(-z[0])))
        assert (np.abs(got_y - y[0]) <= (ey[0] + more * gate) * 1.01 + half * np.abs(y[0]) + 1e-30).all()


@pytest.mark.gpu
@pytest.mark.parametrize("type_", ["f32", "bf16"])
@pytest.mark.parametrize("P", [32, 15])
def test_infinite_gates(gpu_ctx, sampler_lib, type_, P):
    """A gate of -infinity is NaN (-inf / inf in the formula), in prompts and
    steps, and the channels beside it are what they are without it."""
    import torch
    for step in (False, True):
        p, q = (Problem(42, type_, 2, P, 50, 50) for _ in range(2))
        at = torch.zeros(50, p.C, dtype=torch.bool, device="cuda")
        at[::3, ::3] = True
        p.dproj[:, :p.C][at] = -float("inf")
        torch.cuda.synchronize()
        for r in (p, q):
            r.step(sampler_lib, gpu_ctx) if step else r.prefill(sampler_lib, gpu_ctx, [0, 20, 50])
        torch.cuda.synchronize()
        assert p.y[at].isnan().all() and torch.equal(p.y[~at], q.y[~at])
        assert torch.equal(p.dh, q.dh) and torch.equal(p.dconv, q.dconv)


def test_step_refuses_rows_whose_next_overflows(sampler_lib):
    L = sampler_lib.lib()
    ctx = ctypes.create_string_buffer(1 << 16)
    q, most = 1 << 20, 2 ** 31 - 1
    layer = sampler_lib.SsmLayer(1, 1, most, "f32", conv_w=q, conv_b=q, dt_bias=q, a_log=q, d=q, conv_state=q, h_state=q).ref
    assert L.bm_ssm_step(ctx, layer, q, q, q, q, q, 8, most, q, q, 8, None) == -4
    assert L.bm_ssm_step(ctx, layer, q, q, q, q, q, 8, most - 65535, q, q, 8, None) == -4
