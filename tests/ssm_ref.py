"""The state space mixer from its definition in 64 bits, token by token, with
a running bound on what fp32 evaluation may be off by (test infrastructure).

The bound follows the formulas of include/bm_sampler.h with u = 2^-24, first
order in u, counting roundings and the error bounds of the functions called:
  softplus   expf 2 ulp, log1pf 2 ulp, one addition     -> 8 u relative
  a          argument exp(a_log) * softplus: 8 u + expf 4 u + 1 u relative,
             then expf: (13 |arg| + 4) u relative
  g          softplus * B: 9 u relative
  conv       five roundings of the partial sums, each at most the sum of
             magnitudes S: 5 u S
  silu       e^-v by ex2.approx: the rounding of v * log2(e) and 2 ulp,
             (4 + 1.5 |v|) u relative; reciprocal, sum and product 4 u;
             slope at most 1.1 for the error of v
  scan       E_t = a E_{t-1} + err(a) |s_{t-1}| + err(g u) + 2 u (|a s| + |g u|)
             (|s| itself, not the sum of magnitudes: the recurrence is
             evaluated on it), doubled where a kernel may sum it in two parts
  bf16       half a step of the result: eps / 2 = 2^-8 relative
"""
import numpy as np

U = 2.0 ** -24


def _silu(v, ev):
    s = v / (1.0 + np.exp(-v))
    return s, 1.1 * ev + (8.0 + 1.5 * np.abs(v)) * U * np.abs(s)


def run(x, z, b, c, dt, w, H, P, conv, h, fresh):
    """One sequence.  x, z (or None) [T, C], b, c, dt [T, H] float64; w a dict
    of float64 weights; conv [3, C], h [C].  Returns y, ey, conv', h', eh'."""
    T, C = x.shape
    if fresh:
        conv, h = np.zeros_like(conv), np.zeros_like(h)
    win = np.concatenate([conv, x])
    head = np.arange(C) // P
    y, ey = np.empty((T, C)), np.empty((T, C))
    eh, mag = np.zeros(C), np.abs(h)
    for t in range(T):
        terms = win[t:t + 4].T * w["conv_w"]
        v = w["conv_b"] + terms.sum(1)
        u, eu = _silu(v, 5 * U * (np.abs(w["conv_b"]) + np.abs(terms).sum(1)))
        d = np.logaddexp(dt[t] + w["dt_bias"], 0.0)
        arg = np.exp(w["a_log"]) * d
        # the argument of softplus is itself rounded
        ed = 8 * U * d + U * np.abs(dt[t] + w["dt_bias"])
        a = np.exp(-arg)[head]
        ea = ((13 * arg + 4) * U + ed * np.exp(w["a_log"]))[head] * a
        g = (d * b[t])[head]
        eg = 9 * U * np.abs(g) + (ed * np.abs(b[t]))[head]
        # in two parts (a tile's own sum and what came before it) the sums of
        # magnitudes bound both
        mag = a * mag + np.abs(g * u)
        eh = a * eh + ea * mag + eg * np.abs(u) + np.abs(g) * eu + 4 * U * mag
        h = a * h + g * u
        cc = c[t][head]
        o = cc * h + w["d"] * u
        eo = np.abs(cc) * eh + np.abs(w["d"]) * eu + 4 * U * (np.abs(cc) * mag + np.abs(w["d"] * u))
        if z is not None:
            s, es = _silu(z[t], 0.0)
            eo = eo * np.abs(s) + np.abs(o) * es + U * np.abs(o * s)
            o = o * s
        y[t], ey[t] = o, eo
    return y, ey, win[T:T + 3], h, eh


def weights(rng, H, P):
    """Steps of 0.001 to 0.1 and decay rates 1 to 16, as such layers start."""
    C = H * P
    step = np.exp(rng.uniform(np.log(1e-3), np.log(0.1), H))
    f = lambda v: np.ascontiguousarray(v, np.float32)  # noqa: E731
    return {"conv_w": f(0.4 * rng.standard_normal((C, 4))), "conv_b": f(0.1 * rng.standard_normal(C)),
            "dt_bias": f(step + np.log(-np.expm1(-step))), "a_log": f(np.log(rng.uniform(1, 16, H))),
            "d": f(1 + 0.1 * rng.standard_normal(C))}
