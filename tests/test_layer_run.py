"""The layer operators together, as a serving loop uses them: a layer's
projection, mixer and projection (bm_ternary_logits or bm_fp8_logits,
bm_ssm_prefill, bm_ssm_step), the decode loop behind them, samples of one
prompt forked, stopped rows compacted away."""
import ctypes

import numpy as np
import pytest

import ssm_ref
import synth
import ternary

pytestmark = pytest.mark.gpu
DEFAULT = 1


class Block:
    """One layer on the device, ternary or fp8 projections, fp32 states."""

    def __init__(self, bm, ctx, seed, d, H, slots, kind):
        import torch
        self.bm, self.ctx, self.torch, self.kind = bm, ctx, torch, kind
        self.d, self.H, self.C, self.slots = d, H, 2 * d, slots
        self.P, self.rows_in = self.C // H, 2 * self.C + 3 * H
        rng = np.random.default_rng(seed)
        self.w = ssm_ref.weights(rng, H, self.P)
        self.dev = {k: torch.from_numpy(v).cuda() for k, v in self.w.items()}
        self.conv = torch.zeros(slots, 3, self.C, device="cuda")
        self.h = torch.zeros(slots, self.C, device="cuda")
        self.layer = bm.SsmLayer(H, self.P, slots, "f32", **{k: v.data_ptr() for k, v in self.dev.items()},
                                 conv_state=self.conv.data_ptr(), h_state=self.h.data_ptr())
        self.ld = -(-self.rows_in // 8) * 8
        self.norm = [torch.from_numpy((1 + 0.02 * rng.standard_normal(n)).astype(np.float32)).cuda() for n in (d, self.C)]
        self.mats = []
        for n, k in ((self.rows_in, d), (d, self.C)):
            if kind == "ternary":
                codes = synth.ternary_codes(seed + n, 3, n, k)
                pk = torch.from_numpy(np.ascontiguousarray(codes, np.uint8)).cuda()
                w8 = torch.empty(n, k, dtype=torch.int8, device="cuda")
                torch.cuda.synchronize()
                ctx.ternary_unpack(pk.data_ptr(), n, k, w8.data_ptr(), DEFAULT)
                torch.cuda.synchronize()
                self.mats.append((codes, w8))
            else:
                w = torch.from_numpy(rng.standard_normal((n, k)).astype(np.float32) * 60).cuda()
                s = torch.from_numpy((rng.random((-(-n // 128), -(-k // 128))) * 2e-3 + 1e-3).astype(np.float32)).cuda()
                self.mats.append((w.clamp(-448, 448).to(torch.float8_e4m3fn), s))

    def project(self, i, x, out, ld):
        B, k = x.shape
        n = self.rows_in if i == 0 else self.d
        m = self.mats[i]
        if self.kind == "ternary":
            self.ctx.ternary_logits(x.data_ptr(), B, k, None, self.norm[i].data_ptr(), m[1].data_ptr(), 30.0, n,
                                    out.data_ptr(), ld, DEFAULT)
        else:
            self.ctx.fp8_logits(x.data_ptr(), B, k, self.norm[i].data_ptr(), m[0].data_ptr(), m[1].data_ptr(), n,
                                out.data_ptr(), ld, DEFAULT)

    def run(self, x, mix):
        """x + out_proj(mixer(in_proj(x))); mix(ptrs, rows, y) runs the mixer."""
        t = self.torch
        B = x.shape[0]
        proj = t.zeros(B, self.ld, device="cuda")
        y = t.zeros(B, self.C, device="cuda")
        o = t.empty(B, self.d, device="cuda")
        t.cuda.synchronize()
        self.project(0, x, proj, self.ld)
        at, C, H = proj.data_ptr(), self.C, self.H
        mix([at + 4 * C, at, at + 8 * C, at + 4 * (2 * C + H), at + 4 * (2 * C + 2 * H)], B, y)
        self.project(1, y, o, self.d)
        t.cuda.synchronize()
        self.proj, self.y = proj, y
        return x + o

    def prefill(self, x, off, slots, fresh):
        t = self.torch
        a = [t.tensor(off, dtype=t.int64, device="cuda"), t.tensor(slots, dtype=t.int32, device="cuda"),
             t.tensor(fresh, dtype=t.int32, device="cuda")]
        return self.run(x, lambda q, B, y: self.ctx.ssm_prefill(
            self.layer, *q, self.ld, B, a[0].data_ptr(), len(slots), a[1].data_ptr(), a[2].data_ptr(), y.data_ptr(), self.C,
            DEFAULT))

    def step(self, x):
        return self.run(x, lambda q, B, y: self.ctx.ssm_step(self.layer, *q, self.ld, B, None, y.data_ptr(), self.C, DEFAULT))

    def regions(self):
        return self.bm.slot_regions([(self.conv.data_ptr(), 12 * self.C, 12 * self.C, 1, 0),
                                     (self.h.data_ptr(), 4 * self.C, 4 * self.C, 1, 0)])

    def check_mixer(self, off, conv0, h0, fresh):
        """The mixer against its definition on the projection that it got."""
        f = self.proj.double().cpu().numpy()
        C, H = self.C, self.H
        w = {k: v.astype(np.float64) for k, v in self.w.items()}
        for i in range(len(off) - 1):
            r = slice(off[i], off[i + 1])
            y, ey, _, _, _ = ssm_ref.run(f[r, C:2 * C], f[r, :C], *(f[r, 2 * C + k * H:2 * C + (k + 1) * H] for k in range(3)),
                                         w, H, self.P, conv0[i], h0[i], fresh[i])
            got = self.y[r].double().cpu().numpy()
            assert (np.abs(got - y) <= 1.01 * ey + ssm_ref.U * np.abs(y)).all()


@pytest.mark.parametrize("kind", ["ternary", "fp8"])
def test_serving_loop(gpu_ctx, sampler_lib, oracle_lib, kind):
    import torch
    bm, ctx = sampler_lib, gpu_ctx
    d, H, B, V = 128, 4, 6, 1000
    blk = Block(bm, ctx, 5, d, H, B, kind)
    rng = np.random.default_rng(1)
    embed = torch.from_numpy(rng.standard_normal((V, d)).astype(np.float32)).cuda()
    head = torch.from_numpy(rng.standard_normal((V, d)).astype(np.float32)).cuda()
    hw = (head * 40).clamp(-448, 448).to(torch.float8_e4m3fn)
    hs = torch.full((-(-V // 128), 1), 0.002, device="cuda")
    hn = torch.ones(d, device="cuda")

    # the in_proj of the ternary block is the oracle's, bit for bit
    prompts = [list(rng.integers(1, V, n)) for n in (5, 1, 40, 17, 33, 2)]
    off = [0] + list(np.cumsum([len(p) for p in prompts]))
    x = embed[torch.tensor(sum(prompts, []), device="cuda")]
    zero = np.zeros((B, 3, blk.C)), np.zeros((B, blk.C))
    out = blk.prefill(x, off, list(range(B)), [1] * B)
    if kind == "ternary":
        q = ternary.prep(x.cpu().numpy(), None, blk.norm[0].cpu().numpy(), np.float32(30.0))
        want = ternary.logits_fast(*q, blk.mats[0][0])
        assert np.array_equal(blk.proj[:, :blk.rows_in].cpu().numpy(), want)
    blk.check_mixer(off, *zero, [True] * B)

    dec = bm.Decode(ctx, B, max_tokens=0, stop_ids=[])
    dec.reset(prompts)
    kn = bm.knobs_array(0.8, 1.1, 0.0, 0.95, 40)
    kd = torch.from_numpy(kn.view(np.uint8).copy()).cuda()
    last = out[torch.tensor(off[1:], device="cuda") - 1].contiguous()

    def sample(hidden, step, rows):
        logits = torch.empty(rows, V, device="cuda")
        u = torch.from_numpy(synth.uniform(3, 50 + step, rows).astype(np.float32)).cuda()
        ids = torch.empty(rows, dtype=torch.int32, device="cuda")
        hist = dec.read()["ring"][:rows]
        torch.cuda.synchronize()
        ctx.fp8_logits(hidden.data_ptr(), rows, d, hn.data_ptr(), hw.data_ptr(), hs.data_ptr(), V, logits.data_ptr(), V, DEFAULT)
        dec.step(logits.data_ptr(), V, V, kd.data_ptr(), 0, u.data_ptr(), ids.data_ptr(), DEFAULT)
        torch.cuda.synchronize()
        b = synth.Batch(logits.cpu().numpy(), hist.reshape(-1).astype(np.int32), np.arange(rows + 1, dtype=np.int64) * 256,
                        np.full(rows, 0.8, np.float32), np.full(rows, 1.1, np.float32), np.zeros(rows, np.float32),
                        np.full(rows, 0.95, np.float32), np.full(rows, 40, np.int32))
        rids, _, res = oracle_lib.sample_batch(b, u.cpu().numpy())
        import parity
        got = ids.cpu().numpy()
        assert parity.compare(got, None, rids, None, res)["bad"] == 0
        return got

    def step(ids):
        conv0, h0 = blk.conv.double().cpu().numpy(), blk.h.double().cpu().numpy()
        n = len(ids)
        o = blk.step(embed[torch.tensor(ids, device="cuda").long().clamp(min=0)])
        blk.check_mixer(list(range(n + 1)), conv0, h0, [False] * n)
        return o

    ids = sample(last, 0, B)
    hidden = step(ids)
    # three samples of row 2: its loop state and its model state
    src = torch.tensor([0, 2, 2, 3, 2, 5], dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    dec.reorder(src.data_ptr(), blk.regions(), DEFAULT)
    torch.cuda.synchronize()
    for a in (blk.conv, blk.h):
        assert torch.equal(a[1], a[2]) and torch.equal(a[4], a[2])
    ids = sample(hidden[src.long()].contiguous(), 1, B)
    hidden = step(ids)
    # the last row ends; the others go on in fewer rows
    logits = torch.zeros(B, V, device="cuda")
    want = np.array([7, 8, 9, 0, 11, 0])  # token 0 stops a row
    logits[torch.arange(B), torch.from_numpy(want).cuda()] = 50.0
    u, o = torch.zeros(B, device="cuda"), torch.empty(B, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    dec.step(logits.data_ptr(), V, V, kd.data_ptr(), 0, u.data_ptr(), o.data_ptr(), DEFAULT)
    torch.cuda.synchronize()
    assert list(o.cpu().numpy()) == list(want)
    before = blk.h.clone()
    row_of = torch.empty(B, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    dec.compact(blk.regions(), row_of.data_ptr(), DEFAULT)
    torch.cuda.synchronize()
    assert list(row_of.cpu().numpy()) == [0, 1, 2, 4, 3, 5]
    assert torch.equal(blk.h[:4], before[[0, 1, 2, 4]])
    n = dec.active(DEFAULT)
    assert n == 4
    dec.set_rows(n)
    hidden = step([7, 8, 9, 11])
    sample(hidden, 2, n)
    ctx.check()
    dec.close()
