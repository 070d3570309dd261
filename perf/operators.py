"""The operators of policies with memory that this library offers beside its environments, and
the sizes at which their speed is measured.

A policy that acts on partial observations keeps a state per environment and head. Its memory
layer is the gated delta rule: per head, with S the state [key_dim, value_dim],

    S <- exp(g) S      (cleared where an episode begins)
    S <- S + k (beta (v - S^T k))^T
    o  = scale S^T q

Four kinds of work:

  step      one token for every environment, the state advanced in place: what runs beside each
            step of the simulation.
  forward   whole sequences without gradients: values of a rollout, a long recorded episode.
  train     whole sequences and the gradients of every input: what an update of the policy
            runs. Rollouts come time-major, as they are recorded.
  orth      the update of the policy's matrices: a momentum matrix (or several of one shape)
            replaced by a nearly orthogonal one by five Newton-Schulz steps.

Queries and keys are divided by their norms in the operator where `normalize` is set. Queries,
keys and values are views of one projection's output. `resets` is the probability that a token
begins an episode.
"""
import math

import torch

own = False

EPS = 1e-6                                  # of the norms of queries and keys
COEFFICIENTS = (3.4445, -4.7750, 2.0315)    # of the Newton-Schulz step
STEPS = 5
TYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}


def _delta(kind, batch, length, key_heads, value_heads, key_dim, value_dim, dtype, resets=0.0, time_major=False, normalize=True, name=None):
    c = {"kind": kind, "batch": batch, "length": length, "key_heads": key_heads, "value_heads": value_heads, "key_dim": key_dim,
         "value_dim": value_dim, "dtype": dtype, "resets": resets, "time_major": time_major, "normalize": normalize}
    return dict(c, name=name) if name else c


def _orth(count, rows, cols, dtype, name=None):
    c = {"kind": "orth", "count": count, "rows": rows, "cols": cols, "dtype": dtype}
    return dict(c, name=name) if name else c


def listed():
    return [
        # One environment driven from Python: pure call latency.
        _delta("step", 1, 1, 4, 4, 32, 32, "float32", name="step_1"),
        # The headline 4096 environments, an episode ending now and then.
        _delta("step", 4096, 1, 4, 4, 64, 64, "bfloat16", 0.01, name="step_4096"),
        # A wide memory with shared key heads, an odd number of environments.
        _delta("step", 501, 1, 4, 16, 128, 128, "float16", 0.01, name="step_wide_501"),
        # Values of the largest benchmark batch over a short rollout.
        _delta("forward", 16384, 16, 2, 2, 64, 64, "bfloat16", 0.01, True, name="forward_16384x16"),
        # One long recorded episode: few heads, a long axis.
        _delta("forward", 1, 16384, 4, 8, 128, 128, "bfloat16", name="forward_1x16384"),
        # Odd sizes throughout, full precision, raw queries and keys of small norm.
        _delta("forward", 37, 211, 1, 3, 40, 72, "float32", 0.01, normalize=False, name="forward_odd_f32"),
        # The update on a rollout of the headline environments.
        _delta("train", 4096, 32, 4, 4, 64, 64, "bfloat16", 0.015, True, name="train_4096x32"),
        # An update on long episodes with wide heads.
        _delta("train", 2, 4096, 8, 8, 128, 128, "bfloat16", 0.001, name="train_2x4096"),
        # Odd sizes, shared key heads, full precision.
        _delta("train", 19, 333, 2, 4, 24, 48, "float32", 0.01, name="train_odd_f32"),
        # The matrices of a small policy, all of one shape.
        _orth(12, 256, 128, "float32", name="orth_12x256x128"),
        # A wide feed-forward matrix.
        _orth(1, 1000, 4000, "float32", name="orth_1000x4000_f32"),
        # The largest.
        _orth(1, 4096, 4096, "bfloat16", name="orth_4096"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["step", "forward", "train", "orth"])
    if kind == "orth":
        dtype = rng.choice(["float32", "bfloat16", "float16"])
        rows, cols = _log_int(rng, 16, 4096), _log_int(rng, 16, 4096)
        most = max(1, min(16, (1 << 22) // (rows * cols)))
        return _orth(_log_int(rng, 1, most), rows, cols, dtype)
    dtype = rng.choice(["float32", "bfloat16", "bfloat16", "float16"])
    dims = [rng.choice([32, 64, 64, 128]) if rng.random() < 0.6 else _log_int(rng, 8, 128) for _ in range(2)]
    key_heads = rng.randint(1, 8)
    value_heads = key_heads * rng.choice([1, 1, 1, 2, 3])
    resets, normalize = rng.choice([0.0, 0.002, 0.01, 0.03]), rng.random() < 0.75
    state = value_heads * dims[0] * dims[1]
    if kind == "step":
        return _delta(kind, _log_int(rng, 1, min(16384, (1 << 27) // state)), 1, key_heads, value_heads, *dims, dtype, resets, False, normalize)
    tokens = min(1 << 17 if kind == "train" else 1 << 18, (1 << 31 if dtype != "float32" else 1 << 30) // state)  # the largest listed, or less
    length = _log_int(rng, 1, min(16384 if kind == "forward" else 4096, tokens))
    batch = _log_int(rng, 1, max(1, min(16384, tokens // length)))
    return _delta(kind, batch, length, key_heads, value_heads, *dims, dtype, resets, rng.random() < 0.5, normalize)


def work(case):
    s = 4 if case["dtype"] == "float32" else 2
    if case["kind"] == "orth":
        m, n = sorted((case["rows"], case["cols"]))
        return {"bytes": 2 * case["count"] * m * n * s, "flops": case["count"] * STEPS * (m * m * n + m * m * m + 2 * m * m * n)}
    tokens, hk, hv = case["batch"] * case["length"], case["key_heads"], case["value_heads"]
    dk, dv = case["key_dim"], case["value_dim"]
    state = 2 * case["batch"] * hv * dk * dv * 4
    token = (2 * hk * dk + 2 * hv * dv) * s + 8 * hv + 1
    flops = 6 * dk * dv * hv
    if case["kind"] == "train":
        # The gradients of o and of the last state come in, those of every input go out.
        token += (2 * hk * dk + 2 * hv * dv) * s + 8 * hv
        state *= 2
        flops += 14 * dk * dv * hv
    return {"bytes": tokens * token + state, "flops": tokens * flops}


# ---- inputs ----------------------------------------------------------------------------------
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = TYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    if case["kind"] == "orth":
        # A momentum matrix: a few strong directions over noise.
        n, m, k = case["count"], case["rows"], case["cols"]
        r = min(8, m, k)
        x = (0.02 * normal(n, m, k) + normal(n, m, r) @ normal(n, r, k) * (0.3 / math.sqrt(r))) * 1e-3
        return {"case": case, "x": x.to(dtype)}
    b, t, hk, hv, dk, dv = (case[x] for x in ("batch", "length", "key_heads", "value_heads", "key_dim", "value_dim"))
    lead = (t, b) if case["time_major"] else (b, t)

    def batch_first(x):
        return x.transpose(0, 1) if case["time_major"] else x

    x = batch_first(normal(*lead, 2 * hk * dk + hv * dv).to(dtype))
    q, k, v = x.split([hk * dk, hk * dk, hv * dv], -1)
    q, k, v = q.unflatten(-1, (hk, dk)), k.unflatten(-1, (hk, dk)), v.unflatten(-1, (hv, dv))
    if not case["normalize"]:
        q, k = q * dk ** -0.5, k * (0.7 * dk ** -0.5)
    rate = torch.exp(torch.linspace(-5.0, 0.0, hv, device="cuda"))  # heads that forget slowly to fast
    g = batch_first(-rate * torch.nn.functional.softplus(normal(*lead, hv)))
    beta = batch_first(torch.sigmoid(normal(*lead, hv)))
    reset = batch_first(torch.rand(*lead, generator=gen, device="cuda") < case["resets"]) if case["resets"] else None
    state = 0.3 * normal(b, hv, dk, dv)
    s = {"case": case, "q": q, "k": k, "v": v, "g": g, "beta": beta, "reset": reset, "state": state, "scale": dk ** -0.5}
    if case["kind"] == "train":
        s["grads"] = (batch_first(normal(*lead, hv, dv).to(dtype)), 0.1 * normal(b, hv, dk, dv))
        for n in ("q", "k", "v", "g", "beta", "state"):
            s[n] = s[n].detach().requires_grad_()
    return s


def run(s):
    case = s["case"]
    if case["kind"] == "orth":
        if own:
            from zeno_amd.optim import orthogonalize
            return orthogonalize(s["x"], steps=STEPS, coefficients=COEFFICIENTS)
        return _plain_orthogonalize(s["x"])
    inputs = (s["q"], s["k"], s["v"], s["g"], s["beta"])
    if case["kind"] == "step":
        token = [x[:, 0] for x in inputs]
        reset = None if s["reset"] is None else s["reset"][:, 0]
        if own:
            from zeno_amd.memory import gated_delta_step
            o = gated_delta_step(*token, s["state"], reset, scale=s["scale"], normalize=case["normalize"])
        else:
            o = _plain_step(*token, s["state"], reset, s["scale"], case["normalize"])
        return o, s["state"]
    if own:
        from zeno_amd.memory import gated_delta as rule
    else:
        rule = _plain_gated_delta
    if case["kind"] == "forward":
        return rule(*inputs, s["reset"], s["state"], scale=s["scale"], normalize=case["normalize"])
    o, last = rule(*inputs, s["reset"], s["state"], scale=s["scale"], normalize=case["normalize"])
    return (o.detach(), last.detach(), *torch.autograd.grad((o, last), (*inputs, s["state"]), s["grads"]))


# ---- plain forms -----------------------------------------------------------------------------
def _norm(x):
    return x * torch.rsqrt((x * x).sum(-1, keepdim=True) + EPS)


def _plain_step(q, k, v, g, beta, state, reset, scale, normalize):
    dtype, share = q.dtype, v.shape[1] // q.shape[1]
    q, k, v = q.float(), k.float(), v.float()
    if normalize:
        q, k = _norm(q), _norm(k)
    q, k = q.repeat_interleave(share, 1), k.repeat_interleave(share, 1)
    decay = torch.exp(g)
    if reset is not None:
        decay = decay.masked_fill(reset[:, None], 0.0)
    state.mul_(decay[..., None, None])
    u = beta[..., None] * (v - (k[..., None, :] @ state)[..., 0, :])
    state.add_(k[..., :, None] * u[..., None, :])
    return (scale * (q[..., None, :] @ state)[..., 0, :]).to(dtype)


def _unit_lower_inverse(strict):
    """(I + strict)^-1 of strictly lower triangular matrices, by blocks that double in size."""
    n = strict.shape[-1]
    at = torch.arange(n, device=strict.device)
    inv = torch.eye(n, device=strict.device).expand_as(strict)
    size = 1
    while size < n:
        left = (at[:, None] // size == at[None, :] // size + 1) & (at[:, None] // (2 * size) == at[None, :] // (2 * size))
        inv = inv - inv @ (strict * left) @ inv
        size *= 2
    return inv


def _plain_gated_delta(q, k, v, g, beta, reset, state, scale, normalize):
    """The rule over chunks of up to 64 tokens: everything inside the chunks for all of them at
    once, and one loop over the chunks that carries the state."""
    dtype, (b, t, hk, _), hv = q.dtype, q.shape, v.shape[2]
    c = min(64, 1 << max(0, t - 1).bit_length())
    pad = -t % c
    if reset is None:
        reset = torch.zeros(b, t, dtype=torch.bool, device=q.device)

    def chunks(x, heads):  # [b, t, heads, ...] -> [b, hv, chunk, token, ...]
        x = torch.nn.functional.pad(x, (0, 0) * (x.dim() - 2) + (0, pad)).unflatten(1, (-1, c)).movedim(3, 1)
        return x.repeat_interleave(hv // heads, 1) if heads < hv else x

    q, k, v = chunks(q.float(), hk), chunks(k.float(), hk), chunks(v.float(), hv)
    g, beta = chunks(g.masked_fill(reset[..., None], 0.0), hv), chunks(beta, hv)
    episode = chunks(reset[..., None].expand(b, t, hv).float(), hv).cumsum(-1)
    if normalize:
        q, k = _norm(q), _norm(k)
    total = g.cumsum(-1)
    lower = torch.ones(c, c, dtype=torch.bool, device=q.device).tril()
    seen = (episode[..., :, None] == episode[..., None, :]) & lower
    decay = torch.exp((total[..., :, None] - total[..., None, :]).masked_fill(~seen, -math.inf))
    start = torch.exp(total.masked_fill(episode > 0, -math.inf))[..., None]
    kk = (k @ k.transpose(-1, -2) * decay).tril(-1)
    qk = q @ k.transpose(-1, -2) * decay
    inv = _unit_lower_inverse(kk * beta[..., None, :])
    inv_v, inv_k, end = inv @ v, inv @ (start * k), decay[..., -1, :, None]
    states, us = [], []
    for n in range(q.shape[2]):
        u = beta[:, :, n, :, None] * (inv_v[:, :, n] - inv_k[:, :, n] @ state)
        states.append(state)
        us.append(u)
        state = start[:, :, n, -1:] * state + k[:, :, n].transpose(-1, -2) @ (end[:, :, n] * u)
    o = scale * (start * (q @ torch.stack(states, 2)) + qk @ torch.stack(us, 2))
    return o.movedim(1, 3).flatten(1, 2)[:, :t].to(dtype), state


def _plain_orthogonalize(x):
    a, b, c = COEFFICIENTS
    y = x.float()
    if x.shape[-2] > x.shape[-1]:
        y = y.transpose(-1, -2)
    y = y / (torch.sqrt((y * y).sum((-2, -1), keepdim=True)) + 1e-7)
    for _ in range(STEPS):
        gram = y @ y.transpose(-1, -2)
        y = a * y + (b * gram + c * (gram @ gram)) @ y
    return (y.transpose(-1, -2) if x.shape[-2] > x.shape[-1] else y).to(x.dtype)


# ---- the definitions in 64 bits --------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "orth":
        # The other side's products: X (a + b X^T X + c (X^T X)^2), on the smaller one.
        a, b, c = COEFFICIENTS
        x = s["x"].double()
        x = x / (torch.linalg.matrix_norm(x)[:, None, None] + 1e-7)
        for _ in range(STEPS):
            if x.shape[-1] <= x.shape[-2]:
                g = x.mT.contiguous() @ x
                x = a * x + b * (x @ g) + c * ((x @ g) @ g)
            else:
                g = x @ x.mT.contiguous()
                x = a * x + b * (g @ x) + c * (g @ (g @ x))
        return x
    with torch.no_grad():
        return _exact_delta(case, s)


def _exact_delta(case, s):
    """Token by token, and back token by token."""
    share = case["value_heads"] // case["key_heads"]
    q0, k0, v, g, beta = (s[n].detach().double() for n in ("q", "k", "v", "g", "beta"))
    state = s["state"].detach().double()
    rq = rk = None
    if case["normalize"]:
        rq, rk = (1 / (x.square().sum(-1, keepdim=True) + EPS).sqrt() for x in (q0, k0))
    q, k = (x if r is None else x * r for x, r in ((q0, rq), (k0, rk)))
    qh, kh = q.repeat_interleave(share, 2), k.repeat_interleave(share, 2)
    decay = g.exp()
    if s["reset"] is not None:
        decay = torch.where(s["reset"][..., None], torch.zeros_like(decay), decay)
    o, errs, befores = torch.empty_like(v), torch.empty_like(v), []
    for t in range(case["length"]):
        befores.append(state)
        faded = decay[:, t, :, None, None] * state
        errs[:, t] = v[:, t] - (faded * kh[:, t, :, :, None]).sum(-2)
        state = faded + kh[:, t, :, :, None] * (beta[:, t, :, None] * errs[:, t])[:, :, None, :]
        o[:, t] = s["scale"] * (state * qh[:, t, :, :, None]).sum(-2)
        if case["kind"] != "train":
            befores.clear()
    if case["kind"] == "step":
        return o[:, 0], state
    if case["kind"] == "forward":
        return o, state
    do, ds = s["grads"][0].double(), s["grads"][1].double()
    dq, dk, dv, dg, dbeta = torch.empty_like(qh), torch.empty_like(kh), torch.empty_like(v), torch.empty_like(g), torch.empty_like(beta)
    after = state
    for t in reversed(range(case["length"])):
        kt, qt, at = kh[:, t, :, :, None], qh[:, t, :, :, None], decay[:, t, :, None, None]
        before, bt = befores.pop(), beta[:, t, :, None]
        out = s["scale"] * do[:, t][:, :, None, :]
        dq[:, t] = (after * out).sum(-1)
        ds = ds + qt * out
        du = (ds * kt).sum(-2)
        dbeta[:, t] = (du * errs[:, t]).sum(-1)
        derr = bt * du
        dv[:, t] = derr
        faded = at * before
        dk[:, t] = (ds * (bt * errs[:, t])[:, :, None, :]).sum(-1) - (faded * derr[:, :, None, :]).sum(-1)
        ds = ds - kt * derr[:, :, None, :]
        dg[:, t] = (ds * faded).sum((-2, -1))
        ds = at * ds
        after = before
    dq, dk = (x.unflatten(2, (-1, share)).sum(3) for x in (dq, dk))
    if case["normalize"]:
        dq, dk = (r * (d - x * (x * d).sum(-1, keepdim=True)) for r, d, x in ((rq, dq, q), (rk, dk, k)))
    return o, state, dq, dk, dv, dg, dbeta, ds
