"""The model-layer operators beside the sampler: what they compute, in plain
torch operations and through the library, over the sizes they serve.

  prefill   short causal convolution + selective state space scan + gate over
            ragged prompts, continuing or starting the sequences' states
  step      the same for one token per sequence
  reorder   slots of a state cache copied, forked, permuted or compacted in
            place by a row map
  quantize  (RMSNorm and) rounding of activations to 8-bit floats with one
            scale per row and block of 128
  product   8-bit float matrix product with a scale per block of 128 of the
            activations' rows and per 128 x 128 block of the weights

A projection row holds [z | x | B | C | dt]: 2 d_inner + 3 n_heads columns,
the in_proj rows of the packed model file (one B, C and dt per head).
"""
import math
import os
import sys

import torch

own = False

CONV = 4
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
FP8 = torch.float8_e4m3fn
FP8_MAX = 448.0


# ---------------------------------------------------------------- cases --

def listed():
    return [
        # three short prompts arriving together, one with a single token
        dict(name="prefill short", op="prefill", type="f32", rows=48, seqs=3, heads=16, head_dim=64, fresh=1.0),
        # a serving batch's ragged prompts, some of them continued, d_model 2048
        dict(name="prefill ragged", op="prefill", type="f32", rows=4099, seqs=13, heads=32, head_dim=128, fresh=0.6),
        # one long document
        dict(name="prefill long", op="prefill", type="bf16", rows=65536, seqs=1, heads=64, head_dim=64, fresh=1.0),
        # the next token of one conversation
        dict(name="step one", op="step", type="bf16", rows=1, slots=8, heads=32, head_dim=128),
        # a large decode batch over a larger cache
        dict(name="step batch", op="step", type="f32", rows=1024, slots=1280, heads=32, head_dim=128),
        # one prompt's state forked to eight samples of it
        dict(name="reorder fork", op="reorder", kind="fork", type="f32", slots=64, moves=8, layers=24, channels=2048),
        # the live sequences of a large batch moved together
        dict(name="reorder compact", op="reorder", kind="compact", type="f32", slots=1024, moves=512, layers=8, channels=4096),
        # one token's normalised activations
        dict(name="quantize one", op="quantize", type="f32", rows=1, d=2048, norm=True),
        # the out_proj input of a prefill
        dict(name="quantize batch", op="quantize", type="f32", rows=8192, d=4096, norm=False),
        # the lm_head of one token
        dict(name="product one", op="product", rows=1, d=2048, n=50257),
        # an in_proj of a decode batch: 2 * 4096 + 3 * 32 outputs
        dict(name="product in_proj", op="product", rows=72, d=2048, n=8288),
        # the lm_head of a large batch
        dict(name="product lm_head", op="product", rows=2048, d=2048, n=50257),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["prefill", "prefill", "step", "reorder", "quantize", "product", "product"])
    if op in ("prefill", "step"):
        head_dim = rng.choice([16, 24, 32, 40, 64, 64, 80, 96, 128, 128])
        heads = _log(rng, 2, max(2, 4096 // head_dim))
        type_ = rng.choice(["f32", "bf16"])
        if op == "prefill":
            rows = _log(rng, 1, 40000)
            return dict(op=op, type=type_, rows=rows, seqs=_log(rng, 1, max(1, min(200, rows))), heads=heads,
                        head_dim=head_dim, fresh=rng.choice([0.0, 0.5, 1.0]))
        rows = _log(rng, 1, 1024)
        return dict(op=op, type=type_, rows=rows, slots=rows + rng.randrange(0, 64), heads=heads, head_dim=head_dim)
    if op == "reorder":
        slots = _log(rng, 2, 1024)
        return dict(op=op, kind=rng.choice(["fork", "compact", "permute"]), type=rng.choice(["f32", "bf16"]), slots=slots,
                    moves=_log(rng, 1, slots), layers=rng.randrange(1, 9), channels=64 * _log(rng, 2, 64))
    if op == "quantize":
        return dict(op=op, type=rng.choice(["f32", "bf16"]), rows=_log(rng, 1, 8192), d=16 * _log(rng, 8, 256),
                    norm=rng.choice([True, False]))
    return dict(op=op, rows=_log(rng, 1, 2048), d=16 * _log(rng, 8, 256), n=_log(rng, 64, 25000))


# --------------------------------------------------------------- inputs --

def _offsets(case, gen):
    """Ragged sequence offsets that cover all rows; with more than four
    sequences one of them is empty."""
    rows, n = case["rows"], case["seqs"]
    w = torch.rand(n, generator=gen, dtype=torch.float64) + 0.05
    if n > 4:
        w[n // 2] = 0.0
    cut = torch.round(torch.cumsum(w, 0) / w.sum() * rows).long()
    cut[-1] = rows
    return torch.cat([torch.zeros(1, dtype=torch.long), cut])


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    cpu = torch.Generator().manual_seed(seed)
    g = torch.Generator(device=dev).manual_seed(seed)

    def normal(*shape, scale=1.0, dtype=torch.float32):
        return (torch.randn(*shape, generator=g, device=dev) * scale).to(dtype)

    s = dict(case)
    op = case["op"]
    if op in ("prefill", "step"):
        t = TYPES[case["type"]]
        H, P = case["heads"], case["head_dim"]
        C = H * P
        ld = -(-(2 * C + 3 * H) // 8) * 8
        rows = case["rows"]
        s["proj"] = torch.empty(rows, ld, device=dev, dtype=t)
        for r0 in range(0, rows, 8192):
            s["proj"][r0:r0 + 8192] = normal(min(8192, rows - r0), ld, dtype=t)
        s["conv_w"], s["conv_b"] = normal(C, CONV, scale=0.4), normal(C, scale=0.1)
        # steps of 0.001 to 0.1 and decay rates of 1 to 16, as such layers are initialised
        step = torch.exp(torch.rand(H, generator=g, device=dev) * math.log(100.0) + math.log(1e-3))
        s["dt_bias"] = step + torch.log(-torch.expm1(-step))
        s["a_log"] = torch.log(torch.rand(H, generator=g, device=dev) * 15.0 + 1.0)
        s["d"] = 1.0 + normal(C, scale=0.1)
        n = case["seqs"] if op == "prefill" else rows
        slots = n + 3 if op == "prefill" else case["slots"]
        s["conv"] = normal(slots, CONV - 1, C, dtype=t)
        s["h"] = normal(slots, C, scale=0.5)
        s["slots"] = torch.randperm(slots, generator=cpu)[:n].to(torch.int32).to(dev)
        s["y"] = torch.zeros(rows, C, device=dev, dtype=t)
        if op == "prefill":
            s["off"] = _offsets(case, cpu).to(dev)
            s["fresh"] = (torch.rand(n, generator=cpu) < case["fresh"]).to(torch.int32).to(dev)
    elif op == "reorder":
        t = TYPES[case["type"]]
        S, L, C, m = case["slots"], case["layers"], case["channels"], case["moves"]
        s["conv"] = normal(L, S, CONV - 1, C, dtype=t)
        s["h"] = normal(L, S, C)
        src = torch.arange(S)
        pick = torch.randperm(S, generator=cpu)[:m]
        if case["kind"] == "fork":  # m slots take the state of one
            src[pick] = pick[0].clone()
        elif case["kind"] == "permute":
            src[pick] = pick[torch.randperm(m, generator=cpu)]
        else:  # m live slots, in order, to the front
            src[:m] = torch.sort(pick).values
        s["src"] = src.to(torch.int32).to(dev)
    elif op == "quantize":
        t = TYPES[case["type"]]
        # activations with a few large channels
        s["x"] = (normal(case["rows"], case["d"]) * torch.exp(0.5 * normal(case["d"]))).to(t)
        s["w"] = 1.0 + normal(case["d"], scale=0.02) if case["norm"] else None
        s["q"] = torch.empty(case["rows"], case["d"], device=dev, dtype=FP8)
        s["scale"] = torch.zeros(-(-case["d"] // 128), _pitch(case["rows"]), device=dev)
    else:
        M, K, N = case["rows"], case["d"], case["n"]
        KB, NB = -(-K // 128), -(-N // 128)
        s["a"] = (normal(M, K) * 100.0).clamp_(-FP8_MAX, FP8_MAX).to(FP8)
        s["w"] = torch.empty(N, K, device=dev, dtype=FP8)
        for r0 in range(0, N, 8192):
            s["w"][r0:r0 + 8192] = (normal(min(8192, N - r0), K) * 100.0).clamp_(-FP8_MAX, FP8_MAX).to(FP8)
        s["a_scale"] = torch.zeros(KB, _pitch(M), device=dev)
        s["a_scale"][:, :M] = torch.rand(KB, M, generator=g, device=dev) * 0.01 + 0.005
        s["w_scale"] = torch.rand(NB, KB, generator=g, device=dev) * 2e-4 + 1e-4
        s["out"] = torch.empty(M, N, device=dev)
    return s


def _pitch(rows):
    return -(-rows // 4) * 4


def _split(proj, H, C):
    return proj[:, :C], proj[:, C:2 * C], proj[:, 2 * C:2 * C + H], proj[:, 2 * C + H:2 * C + 2 * H], proj[:, 2 * C + 2 * H:2 * C + 3 * H]


# ----------------------------------------------------------- plain forms --

def _silu(v):
    return v / (1.0 + torch.exp(-v))


def _softplus(v):
    return torch.clamp(v, min=0.0) + torch.log1p(torch.exp(-torch.abs(v)))


def _sequence_rows(off, rows):
    """Each row's sequence and its place in it."""
    t = torch.arange(rows, device=off.device)
    sid = torch.searchsorted(off, t, right=True) - 1
    return t, sid, t - off[sid]


def _conv_input(x, conv, slots, fresh, sid, pos, back):
    """The input `back` tokens before each row: the row above, or the state."""
    shifted = torch.cat([x.new_zeros(min(back, x.shape[0]), x.shape[1]), x[:x.shape[0] - back]])
    old = torch.nonzero((pos < back) & (fresh[sid] == 0)).flatten()
    shifted = torch.where((pos >= back)[:, None], shifted, torch.zeros((), device=x.device, dtype=x.dtype))
    shifted[old] = conv[slots[sid[old]].long(), CONV - 1 - back + pos[old]].to(x.dtype)
    return shifted


def _conv_state_after(x, conv, slots, fresh, off):
    """The last three inputs of each sequence, older ones from the state."""
    n = off[1:] - off[:-1]
    place = n[:, None] + torch.arange(-(CONV - 1), 0, device=x.device)
    old = conv[slots.long()]
    old = torch.where((fresh == 0)[:, None, None], old, torch.zeros_like(old))
    i = torch.arange(slots.numel(), device=x.device)[:, None]
    before = old[i, (place + CONV - 1).clamp(0, CONV - 2)]
    inside = x[(off[:-1, None] + place).clamp(0, x.shape[0] - 1)].to(conv.dtype)
    return torch.where((place >= 0)[:, :, None], inside, before)


def _plain_prefill(s):
    H, P, rows = s["heads"], s["head_dim"], s["rows"]
    C, Q = H * P, 128
    z, x, b, c, dt = (v.float() for v in _split(s["proj"], H, C))
    off, slots, fresh = s["off"], s["slots"], s["fresh"]
    t, sid, pos = _sequence_rows(off, rows)
    u = s["conv_b"] + sum(s["conv_w"][:, CONV - 1 - k] * (_conv_input(x, s["conv"], slots, fresh, sid, pos, k) if k else x)
                          for k in range(CONV))
    u = _silu(u)
    step = _softplus(dt + s["dt_bias"])
    cum = torch.cumsum((-torch.exp(s["a_log"]) * step).double(), 0)  # log decay from row 0: a long sum
    before = torch.where(off[:-1, None] > 0, cum[(off[:-1] - 1).clamp(min=0, max=rows - 1)], torch.zeros((), device=u.device, dtype=cum.dtype))
    h0 = torch.where((fresh == 0)[:, None], s["h"][slots.long()], torch.zeros((), device=u.device))
    # chunks of Q rows: [H, K, Q, ...]
    K = -(-rows // Q)
    pad = K * Q - rows

    def chunks(v, fill=0.0):
        return torch.nn.functional.pad(v, (0, 0, 0, pad), value=fill)

    last = (torch.arange(1, K + 1, device=u.device) * Q - 1).clamp(max=rows - 1)
    sidc = torch.nn.functional.pad(sid, (0, pad), value=-1).view(K, Q)
    cumc = chunks(cum).view(K, Q, H).permute(2, 0, 1)
    gc = chunks(step * b).view(K, Q, H).permute(2, 0, 1)
    uc = chunks(u).view(K, Q, H, P).permute(2, 0, 1, 3)
    lower = torch.ones(Q, Q, device=u.device, dtype=torch.bool).tril()
    same = (sidc[:, :, None] == sidc[:, None, :]) & lower
    diff = (cumc[:, :, :, None] - cumc[:, :, None, :]).float()
    weight = torch.exp(torch.where(same, diff, torch.full((), -math.inf, device=u.device))) * gc[:, :, None, :]
    local = weight @ uc  # the state of each row from its chunk alone
    del weight, diff
    # states handed on at the chunks' ends
    end = local.reshape(H, K * Q, P)[:, last]
    cume = cum[last].T
    j, k = torch.arange(K, device=u.device)[None, :], torch.arange(K, device=u.device)[:, None]
    handed = (j < k) & (sid[last][None, :] == sidc[:, 0][:, None])
    diff = (cume[:, (k[:, 0] - 1).clamp(min=0)][:, :, None] - cume[:, None, :]).float()
    carry = torch.exp(torch.where(handed, diff, torch.full((), -math.inf, device=u.device))) @ end
    came = (sidc == sidc[:, :1])
    came[0] = False
    cumk = torch.cat([cum.new_zeros(H, 1), cume[:, :-1]], 1)
    factor = torch.where(came, torch.exp((cumc - cumk[:, :, None]).clamp(max=0.0).float()), torch.zeros((), device=u.device))
    local += factor[..., None] * carry[:, :, None, :]
    h = local.reshape(H, K * Q, P)[:, :rows].permute(1, 0, 2)
    h = h + torch.exp((cum - before[sid]).float())[:, :, None] * h0.view(-1, H, P)[sid]
    y = ((c[:, :, None] * h).reshape(rows, C) + s["d"] * u) * _silu(z)
    ends = off[1:] - 1
    some = (off[1:] > off[:-1])[:, None]
    h_new = torch.where(some, h.reshape(rows, C)[ends.clamp(min=0)], h0)
    conv_new = _conv_state_after(x, s["conv"], slots, fresh, off)
    s["y"].copy_(y)
    s["h"][slots.long()] = h_new
    s["conv"][slots.long()] = conv_new
    return {"y": s["y"], "h": s["h"], "conv": s["conv"]}


def _plain_step(s):
    H, P = s["heads"], s["head_dim"]
    C = H * P
    z, x, b, c, dt = (v.float() for v in _split(s["proj"], H, C))
    at = s["slots"].long()
    old = s["conv"][at]
    window = torch.cat([old.float(), x[:, None]], 1)
    u = _silu(s["conv_b"] + (window * s["conv_w"].T).sum(1))
    step = _softplus(dt + s["dt_bias"])
    a = torch.exp(-torch.exp(s["a_log"]) * step)
    h = a.repeat_interleave(P, 1) * s["h"][at] + (step * b).repeat_interleave(P, 1) * u
    y = (c.repeat_interleave(P, 1) * h + s["d"] * u) * _silu(z)
    s["y"].copy_(y)
    s["h"][at] = h
    s["conv"][at] = torch.cat([old[:, 1:], x[:, None].to(old.dtype)], 1)
    return {"y": s["y"], "h": s["h"], "conv": s["conv"]}


def _plain_reorder(s):
    src = s["src"].long()
    s["conv"].copy_(s["conv"][:, src])
    s["h"].copy_(s["h"][:, src])
    return {"conv": s["conv"], "h": s["h"]}


def _blocks(x):
    rows, d = x.shape
    return torch.nn.functional.pad(x, (0, -d % 128)).view(rows, -1, 128)


def _plain_quantize(s):
    x = s["x"].float()
    rows, d = x.shape
    if s["w"] is not None:
        x = x * (1.0 / torch.sqrt((x * x).mean(1, keepdim=True) + 1e-6)) * s["w"]
    x = _blocks(x)
    top = x.abs().amax(2)
    scale = torch.where(top > 2.0 ** -100, top / FP8_MAX, torch.ones((), device=x.device))
    s["q"].copy_((x / scale[:, :, None]).reshape(rows, -1)[:, :d].to(FP8))
    s["scale"][:, :rows] = scale.T
    return {"q": s["q"], "scale": s["scale"]}


def _plain_product(s):
    a, w = s["a"], s["w"]
    M, K, N = s["rows"], s["d"], s["n"]
    a = a.float() * s["a_scale"][:, :M].T.repeat_interleave(128, 1)[:, :K]
    w = w.float() * s["w_scale"].repeat_interleave(128, 0)[:N].repeat_interleave(128, 1)[:, :K]
    s["out"].copy_(a @ w.T)
    return s["out"]


# ------------------------------------------------------------ the library --

_LIBRARY = {}


def _library():
    """The library's binding, one context per device, and the stream that
    torch works on (handle 1 names the default stream)."""
    dev = torch.cuda.current_device()
    if dev not in _LIBRARY:
        path = os.path.join(os.getcwd(), "bitmamba.c_b200", "python")
        if path not in sys.path:
            sys.path.insert(0, path)
        import bmsampler
        _LIBRARY[dev] = (bmsampler, bmsampler.Context(dev))
    return (*_LIBRARY[dev], torch.cuda.current_stream().cuda_stream or 1)


def _layer(bm, s):
    """The layer's description, made once as a user's program does."""
    if "layer" not in s:
        s["layer"] = bm.SsmLayer(s["heads"], s["head_dim"], s["h"].shape[0], s["type"], conv_w=s["conv_w"].data_ptr(),
                                 conv_b=s["conv_b"].data_ptr(), dt_bias=s["dt_bias"].data_ptr(), a_log=s["a_log"].data_ptr(),
                                 d=s["d"].data_ptr(), conv_state=s["conv"].data_ptr(), h_state=s["h"].data_ptr())
    return s["layer"]


def _own(s):
    bm, ctx, stream = _library()
    op = s["op"]
    if op in ("prefill", "step"):
        layer = _layer(bm, s)
        p, H = s["proj"], s["heads"]
        C, e, at = H * s["head_dim"], p.element_size(), p.data_ptr()
        z, x, b, c, dt = at, at + C * e, at + 2 * C * e, at + (2 * C + H) * e, at + (2 * C + 2 * H) * e
        if op == "prefill":
            ctx.ssm_prefill(layer, x, z, b, c, dt, p.shape[1], s["rows"], s["off"].data_ptr(), s["seqs"],
                            s["slots"].data_ptr(), s["fresh"].data_ptr(), s["y"].data_ptr(), C, stream)
        else:
            ctx.ssm_step(layer, x, z, b, c, dt, p.shape[1], s["rows"], s["slots"].data_ptr(), s["y"].data_ptr(), C, stream)
        return {"y": s["y"], "h": s["h"], "conv": s["conv"]}
    if op == "reorder":
        if "regions" not in s:
            s["regions"] = bm.slot_regions([(v.data_ptr(), v.stride(1) * v.element_size(), v.stride(1) * v.element_size(),
                                             v.shape[0], v.stride(0) * v.element_size()) for v in (s["conv"], s["h"])])
        ctx.slots_reorder(s["regions"], s["src"].data_ptr(), s["slots"], stream)
        return {"conv": s["conv"], "h": s["h"]}
    if op == "quantize":
        ctx.fp8_quantize(s["x"].data_ptr(), s["type"], s["rows"], s["d"], s["d"], s["w"].data_ptr() if s["w"] is not None else None,
                         s["q"].data_ptr(), s["scale"].data_ptr(), s["scale"].shape[1], stream)
        return {"q": s["q"], "scale": s["scale"]}
    ctx.fp8_product(s["a"].data_ptr(), s["a_scale"].data_ptr(), s["a_scale"].shape[1], s["rows"], s["d"], s["w"].data_ptr(),
                    s["w_scale"].data_ptr(), s["n"], s["out"].data_ptr(), s["n"], stream)
    return s["out"]


def run(state):
    if own:
        return _own(state)
    return {"prefill": _plain_prefill, "step": _plain_step, "reorder": _plain_reorder, "quantize": _plain_quantize,
            "product": _plain_product}[state["op"]](state)


def work(case):
    op = case["op"]
    if op in ("prefill", "step"):
        e = 4 if case["type"] == "f32" else 2
        H, rows = case["heads"], case["rows"]
        C = H * case["head_dim"]
        n = case["seqs"] if op == "prefill" else rows
        read = n if op == "step" else n * (1.0 - case["fresh"])
        state = C * (4 + (CONV - 1) * e)
        return {"bytes": rows * (3 * C + 3 * H) * e + (read + n) * state + C * 4 * (CONV + 2), "flops": 30.0 * rows * C}
    if op == "reorder":
        e = 4 if case["type"] == "f32" else 2
        row = case["layers"] * case["channels"] * (4 + (CONV - 1) * e)
        m = case["moves"]
        reads = 1 if case["kind"] == "fork" else m
        return {"bytes": float((reads + max(1, m - 1)) * row), "flops": 0.0}
    if op == "quantize":
        e = 4 if case["type"] == "f32" else 2
        return {"bytes": case["rows"] * (case["d"] * (e + 1) + 4.0 * -(-case["d"] // 128)), "flops": 5.0 * case["rows"] * case["d"]}
    M, K, N = case["rows"], case["d"], case["n"]
    return {"bytes": float(M * K + N * K + 4 * M * N + 4 * -(-K // 128) * (M + -(-N // 128))), "flops": 2.0 * M * N * K}


# ------------------------------------------------ the definitions, 64 bits --

def exact(case, seed):
    """Each operator from its definition in 64 bits: the scan by doubling the
    distance over which rows are combined, the rest element by element."""
    s = prepare(case, seed)
    op = case["op"]
    if op in ("prefill", "step"):
        H, P, rows = case["heads"], case["head_dim"], case["rows"]
        C = H * P
        proj = s["proj"].double()
        dev = proj.device
        off = s["off"] if op == "prefill" else torch.arange(rows + 1, device=dev)
        fresh = s["fresh"].bool() if op == "prefill" else torch.zeros(rows, dtype=torch.bool, device=dev)
        slots = s["slots"].long()
        length = off[1:] - off[:-1]
        sid = torch.repeat_interleave(torch.arange(length.numel(), device=dev), length)
        start = off[:-1][sid]
        conv, h = s["conv"].double(), s["h"].double()
        h0 = h[slots] * (~fresh)[:, None]
        # the inputs of every sequence behind its three old ones, one below the other
        x = proj[:, C:2 * C]
        place = torch.arange(rows, device=dev) + 3 * (sid + 1)
        tall = torch.zeros(rows + 3 * length.numel(), C, device=dev, dtype=torch.float64)
        tall[place] = x
        head = off[:-1] + 3 * torch.arange(length.numel(), device=dev)
        for k in range(CONV - 1):
            tall[head + k] = conv[slots, k] * (~fresh)[:, None]
        u = s["conv_b"].double().expand(rows, C).clone()
        for k in range(CONV):
            u += s["conv_w"][:, k].double() * tall[place - (CONV - 1 - k)]
        u *= torch.sigmoid(u)
        tail = off[1:] + 3 * torch.arange(length.numel(), device=dev)
        conv[slots] = torch.stack([tall[tail + k] for k in range(CONV - 1)], 1)
        del tall
        b, c, dt = (proj[:, 2 * C + k * H:2 * C + (k + 1) * H] for k in range(3))
        step = torch.logaddexp(dt + s["dt_bias"].double(), torch.zeros((), device=dev, dtype=torch.float64))
        a = torch.exp(-torch.exp(s["a_log"].double()) * step)
        v = ((step * b)[:, :, None] * u.view(rows, H, P))
        first = torch.arange(rows, device=dev) == start
        v[first] += a[first][:, :, None] * h0.view(-1, H, P)[sid[first]]
        a[first] = 0.0
        far = 1
        while far < rows:
            v[far:] += a[far:, :, None] * v[:-far].clone()
            a[far:] *= a[:-far].clone()
            far *= 2
        y = (c[:, :, None] * v).reshape(rows, C) + s["d"].double() * u
        z = proj[:, :C]
        y *= z * torch.sigmoid(z)
        h[slots] = torch.where((length > 0)[:, None], v.reshape(rows, C)[(off[1:] - 1).clamp(min=0)], h0)
        return {"y": y, "h": h, "conv": conv}
    if op == "reorder":
        src = s["src"].long()
        return {"conv": torch.stack([v.index_select(0, src) for v in s["conv"]]).double(),
                "h": torch.stack([v.index_select(0, src) for v in s["h"]]).double()}
    if op == "quantize":
        x = s["x"].double()
        if s["w"] is not None:
            x = x / torch.sqrt(x.square().sum(1, keepdim=True) / case["d"] + 1e-6) * s["w"].double()
        scale = torch.zeros(s["scale"].shape, device=x.device, dtype=torch.float64)
        q = torch.empty_like(x)
        for k in range(scale.shape[0]):
            part = x[:, 128 * k:128 * (k + 1)]
            top = part.abs().amax(1)
            scale[k, :case["rows"]] = torch.where(top > 2.0 ** -100, top / FP8_MAX, torch.ones_like(top))
            # rounding to 3 bits behind the leading one, steps of 2^-9 below 2^-6
            v = part / scale[k, :case["rows"], None]
            grid = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)
            q[:, 128 * k:128 * (k + 1)] = torch.round(v / grid) * grid
        return {"q": q, "scale": scale}
    M, K, N = case["rows"], case["d"], case["n"]
    out = torch.zeros(M, N, device=s["a"].device, dtype=torch.float64)
    for k in range(s["a_scale"].shape[0]):
        cut = slice(128 * k, min(K, 128 * (k + 1)))
        w = s["w"][:, cut].double() * s["w_scale"][:, k].double().repeat_interleave(128)[:N, None]
        out += (s["a"][:, cut].double() * s["a_scale"][k, :M, None].double()) @ w.T
    return out
