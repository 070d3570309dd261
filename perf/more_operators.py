"""The layers of a policy's block around its memory, and the sizes at which their speed is measured.

A block normalises its features, passes them through a memory layer, normalises each head's output
and adds the result to its stream of features. Beside the gated delta rule the memory layer may be
linear attention with a decay for each head: per sequence (environment) and head, with S the state
[key_dim, value_dim],

    S <- exp(g) S + k v^T      (S <- k v^T where an episode begins)
    o  = scale S^T q

and the norm of a row x of n features is

    y = (x - mean) / sqrt(variance + eps) * weight + bias

where x may be the sum of a residual stream and what is added to it, which is rounded to its type
and returned too. Five kinds of work:

  step        linear attention, one token for every environment, the state advanced in place: what
              runs beside each step of the simulation.
  forward     whole sequences without gradients: values of a rollout, a long recorded episode.
  train       whole sequences and the gradients of every input, of the decays too where they are
              learned. Rollouts come time-major, as they are recorded.
  norm        rows normalised.
  norm_train  the same with the gradients of the rows, the weight and the bias.

Queries, keys and values are views of one projection's output. `resets` is the probability that a
token begins an episode. Where `view` is set the rows of a norm are part of wider rows.
"""
import math

import torch

own = False

EPS = 1e-5  # of the norm
TYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}


def _linear(kind, batch, length, key_heads, value_heads, key_dim, value_dim, dtype, resets=0.0, time_major=False, learned=False, name=None):
    c = {"kind": kind, "batch": batch, "length": length, "key_heads": key_heads, "value_heads": value_heads, "key_dim": key_dim,
         "value_dim": value_dim, "dtype": dtype, "resets": resets, "time_major": time_major, "learned": learned}
    return dict(c, name=name) if name else c


def _norm(kind, rows, dim, dtype, weights, residual=False, view=False, name=None):
    c = {"kind": kind, "rows": rows, "dim": dim, "dtype": dtype, "weights": weights, "residual": residual, "view": view}
    return dict(c, name=name) if name else c


def listed():
    return [
        # One environment driven from Python: pure call latency.
        _linear("step", 1, 1, 4, 4, 32, 32, "float32", name="step_1"),
        # The headline 4096 environments, an episode ending now and then.
        _linear("step", 4096, 1, 4, 4, 64, 64, "bfloat16", 0.01, name="step_4096"),
        # Values of the largest benchmark batch over a short rollout.
        _linear("forward", 16384, 16, 2, 2, 64, 64, "bfloat16", 0.01, True, name="forward_16384x16"),
        # One long recorded episode: few heads, a long axis.
        _linear("forward", 1, 16384, 4, 8, 128, 128, "float16", name="forward_1x16384"),
        # The update on a rollout of the headline environments, decays fixed.
        _linear("train", 4096, 32, 4, 4, 64, 64, "bfloat16", 0.015, True, name="train_4096x32"),
        # An update on long episodes with wide heads, decays learned.
        _linear("train", 2, 4096, 8, 8, 128, 128, "bfloat16", 0.001, learned=True, name="train_2x4096"),
        # Odd sizes, shared key heads, full precision, decays learned.
        _linear("train", 19, 333, 2, 4, 24, 48, "float32", 0.01, learned=True, name="train_odd_f32"),
        # The features of one environment: pure call latency.
        _norm("norm", 1, 256, "float32", "float32", name="norm_1"),
        # The heads' outputs of a rollout of the headline environments (4096 x 32 tokens, 4 heads).
        _norm("norm", 524288, 64, "bfloat16", "bfloat16", name="norm_heads"),
        # The update on that rollout: the features of a block, added to their stream.
        _norm("norm_train", 131072, 512, "bfloat16", "float32", True, name="norm_train_131072x512"),
        # Odd sizes, full precision.
        _norm("norm_train", 4099, 1000, "float32", "float32", name="norm_train_odd_f32"),
        # Few wide rows of an odd length, part of wider ones.
        _norm("norm_train", 301, 8191, "float16", "float16", view=True, name="norm_train_wide"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["step", "forward", "train", "norm", "norm_train"])
    dtype = rng.choice(["float32", "bfloat16", "bfloat16", "float16"])
    if kind.startswith("norm"):
        dim = rng.choice([32, 64, 128, 256, 512, 1024, 2048]) if rng.random() < 0.4 else _log_int(rng, 8, 8192)
        most = (1 << 26 if kind == "norm_train" else 1 << 25) // dim
        return _norm(kind, _log_int(rng, 1, min(most, 1 << 20)), dim, dtype, rng.choice(["float32", dtype]), rng.random() < 0.4, rng.random() < 0.3)
    dims = [rng.choice([32, 64, 64, 128]) if rng.random() < 0.6 else _log_int(rng, 8, 128) for _ in range(2)]
    key_heads = rng.randint(1, 8)
    value_heads = key_heads * rng.choice([1, 1, 1, 2, 3])
    resets, learned = rng.choice([0.0, 0.002, 0.01, 0.03]), rng.random() < 0.6
    state = value_heads * dims[0] * dims[1]
    if kind == "step":
        return _linear(kind, _log_int(rng, 1, min(16384, (1 << 26) // state)), 1, key_heads, value_heads, *dims, dtype, resets)
    tokens = min(1 << 17 if kind == "train" else 1 << 18, (1 << 31 if dtype != "float32" else 1 << 30) // state)  # the largest listed, or less
    length = _log_int(rng, 1, min(16384 if kind == "forward" else 4096, tokens))
    batch = _log_int(rng, 1, max(1, min(16384, tokens // length)))
    return _linear(kind, batch, length, key_heads, value_heads, *dims, dtype, resets, rng.random() < 0.5, kind == "train" and learned)


def work(case):
    s = 4 if case["dtype"] == "float32" else 2
    if case["kind"].startswith("norm"):
        rows, n = case["rows"], case["dim"]
        passes = 4 if case["residual"] else 2  # x and the stream in, the norm and the stream out
        w, flops = 2 * n * (4 if case["weights"] == "float32" else s), 8 * rows * n
        if case["kind"] == "norm_train":  # the gradients of both come in, that of the rows and the weights' go out
            passes, w, flops = passes + (3 if case["residual"] else 2), 2 * w, flops + 14 * rows * n
        return {"bytes": passes * rows * n * s + w, "flops": flops}
    tokens, hk, hv = case["batch"] * case["length"], case["key_heads"], case["value_heads"]
    dk, dv = case["key_dim"], case["value_dim"]
    state = 2 * case["batch"] * hv * dk * dv * 4
    token = (2 * hk * dk + 2 * hv * dv) * s + (1 if case["resets"] else 0)
    flops = 4 * dk * dv * hv
    if case["kind"] == "train":
        # The gradients of o and of the last state come in, those of every input go out.
        token += (2 * hk * dk + 2 * hv * dv) * s
        state *= 2
        flops += 10 * dk * dv * hv
    return {"bytes": tokens * token + state + 4 * hv, "flops": tokens * flops}


# ---- inputs ----------------------------------------------------------------------------------
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = TYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    if case["kind"].startswith("norm"):
        rows, n = case["rows"], case["dim"]
        columns = (0.5 * normal(n), torch.exp(0.3 * normal(n)))  # features that are off zero and of unlike size

        def features(scale):
            wide = torch.empty(rows, n + 64, dtype=dtype, device="cuda") if case["view"] else None
            x = torch.addcmul(columns[0] * scale, normal(rows, n), columns[1] * scale).to(dtype)
            return wide[:, 32:32 + n].copy_(x) if case["view"] else x

        weights = TYPES[case["weights"]]
        s = {"case": case, "x": features(1.0), "residual": features(2.0) if case["residual"] else None,
             "weight": (1.0 + 0.2 * normal(n)).to(weights), "bias": (0.1 * normal(n)).to(weights)}
        if case["kind"] == "norm_train":
            s["grads"] = tuple(normal(rows, n).to(dtype) for _ in range(2 if case["residual"] else 1))
            for name in ("x", "residual", "weight", "bias"):
                if s[name] is not None:
                    s[name] = s[name].detach().requires_grad_()
        return s
    b, t, hk, hv, dk, dv = (case[x] for x in ("batch", "length", "key_heads", "value_heads", "key_dim", "value_dim"))
    lead = (t, b) if case["time_major"] else (b, t)

    def batch_first(x):
        return x.transpose(0, 1) if case["time_major"] else x

    x = batch_first(normal(*lead, 2 * hk * dk + hv * dv).to(dtype))
    q, k, v = x.split([hk * dk, hk * dk, hv * dv], -1)
    q, k, v = q.unflatten(-1, (hk, dk)), k.unflatten(-1, (hk, dk)), v.unflatten(-1, (hv, dv))
    # Heads that forget slowly to fast.
    g = -torch.exp(torch.linspace(-5.0, 0.0, hv, device="cuda") + 0.2 * normal(hv))
    reset = batch_first(torch.rand(*lead, generator=gen, device="cuda") < case["resets"]) if case["resets"] else None
    state = normal(b, hv, dk, dv)
    s = {"case": case, "q": q, "k": k, "v": v, "g": g, "reset": reset, "state": state, "scale": dk ** -0.5}
    if case["kind"] == "train":
        s["grads"] = (batch_first(normal(*lead, hv, dv).to(dtype)), 0.1 * normal(b, hv, dk, dv))
        for n in ("q", "k", "v", "state") + (("g",) if case["learned"] else ()):
            s[n] = s[n].detach().requires_grad_()
    return s


def run(s):
    case = s["case"]
    if case["kind"].startswith("norm"):
        if not own:
            return _plain_norm(s["x"], s["weight"], s["bias"], s["residual"], s.get("grads"))
        from zeno_amd.norm import layer_norm
        y = layer_norm(s["x"], s["weight"], s["bias"], residual=s["residual"], eps=EPS)
        if case["kind"] == "norm":
            return y
        y = y if case["residual"] else (y,)
        inputs = (s["x"], s["weight"], s["bias"]) + ((s["residual"],) if case["residual"] else ())
        return (*(z.detach() for z in y), *torch.autograd.grad(y, inputs, s["grads"]))
    inputs = (s["q"], s["k"], s["v"], s["g"])
    if case["kind"] == "step":
        token = [x[:, 0] for x in inputs[:3]]
        reset = None if s["reset"] is None else s["reset"][:, 0]
        if own:
            from zeno_amd.memory import linear_attention_step
            o = linear_attention_step(*token, s["g"], s["state"], reset, scale=s["scale"])
        else:
            o = _plain_step(*token, s["g"], s["state"], reset, s["scale"])
        return o, s["state"]
    if own:
        from zeno_amd.memory import linear_attention as rule
    else:
        rule = _plain_linear_attention
    o, last = rule(*inputs, s["reset"], s["state"], scale=s["scale"])
    if case["kind"] == "forward":
        return o, last
    wanted = (s["q"], s["k"], s["v"], s["state"]) + ((s["g"],) if case["learned"] else ())
    return (o.detach(), last.detach(), *torch.autograd.grad((o, last), wanted, s["grads"]))


# ---- plain forms -----------------------------------------------------------------------------
def _plain_norm(x, weight, bias, residual, grads):
    dtype = x.dtype
    with torch.no_grad():
        stream = x if residual is None else (x.float() + residual.float()).to(dtype)
        s, w = stream.float(), weight.float()
        s = s - s.mean(-1, keepdim=True)
        r = torch.rsqrt((s * s).mean(-1, keepdim=True) + EPS)
        unit = s * r
        y = (unit * w + bias.float()).to(dtype)
        out = (y,) if residual is None else (y, stream)
        if grads is None:
            return out if residual is not None else y
        dy = grads[0].float()
        d = dy * w
        dx = r * (d - d.mean(-1, keepdim=True) - unit * (d * unit).mean(-1, keepdim=True))
        if residual is not None:
            dx = dx + grads[1].float()
        dx = dx.to(dtype)
        out += (dx, (dy * unit).sum(0).to(weight.dtype), dy.sum(0).to(bias.dtype))
        return out if residual is None else (*out, dx)


def _plain_step(q, k, v, g, state, reset, scale):
    dtype, share = q.dtype, v.shape[1] // q.shape[1]
    q, k, v = q.float().repeat_interleave(share, 1), k.float().repeat_interleave(share, 1), v.float()
    decay = torch.exp(g).expand(v.shape[:2])
    if reset is not None:
        decay = decay.masked_fill(reset[:, None], 0.0)
    state.mul_(decay[..., None, None]).add_(k[..., :, None] * v[..., None, :])
    return (scale * (q[..., None, :] @ state)[..., 0, :]).to(dtype)


def _plain_linear_attention(q, k, v, g, reset, state, scale):
    """Chunks of up to 64 tokens: everything inside the chunks for all of them at once, and one
    loop over the chunks that carries the state."""
    dtype, (b, t, hk, _), hv = q.dtype, q.shape, v.shape[2]
    c = min(64, 1 << max(0, t - 1).bit_length())
    pad = -t % c
    if reset is None:
        reset = torch.zeros(b, t, dtype=torch.bool, device=q.device)

    def chunks(x, heads):  # [b, t, heads, n] -> [b, hv, chunk, token, n]
        x = torch.nn.functional.pad(x, (0, 0, 0, 0, 0, pad)).unflatten(1, (-1, c)).movedim(3, 1)
        return x.repeat_interleave(hv // heads, 1) if heads < hv else x

    q, k, v = chunks(q.float(), hk), chunks(k.float(), hk), chunks(v.float(), hv)
    at = torch.arange(c, device=q.device)
    apart = at[:, None] - at[None, :]
    episode = torch.nn.functional.pad(reset, (0, pad)).unflatten(1, (-1, c)).cumsum(-1)[:, None]  # [b, 1, chunk, token]
    seen = (episode[..., :, None] == episode[..., None, :]) & (apart >= 0)
    qk = q @ k.transpose(-1, -2) * (torch.exp(g[:, None, None] * apart.clamp(min=0))[:, None] * seen)
    start = torch.exp(g[:, None] * (at + 1.0))[:, None] * (episode == 0)
    # What is left of each token, and of the state before the chunk, behind its last token.
    length = torch.full((q.shape[2],), c, device=q.device)
    length[-1] = c - pad
    end = torch.exp(g[:, None, None] * (length[:, None] - 1.0 - at).clamp(min=0.0)) * (episode == episode[..., -1:])
    through = torch.exp(g[:, None] * length) * (episode[..., -1] == 0)
    added = (k * end[..., None]).transpose(-1, -2) @ v
    states = []
    for n in range(q.shape[2]):
        states.append(state)
        state = through[:, :, n, None, None] * state + added[:, :, n]
    o = scale * (start[..., None] * (q @ torch.stack(states, 2)) + qk @ v)
    return o.movedim(1, 3).flatten(1, 2)[:, :t].to(dtype), state


# ---- the definitions in 64 bits --------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return _exact_norm(case, s) if case["kind"].startswith("norm") else _exact_linear(case, s)


def _exact_norm(case, s):
    x = s["x"].double()
    if case["residual"]:
        x = (x + s["residual"].double()).to(s["x"].dtype)  # the stream, as its type holds it
    stream, x, w = x, x.double(), s["weight"].double()
    variance, mean = torch.var_mean(x, -1, correction=0, keepdim=True)
    root = torch.sqrt(variance + EPS)
    y = (x - mean) / root * w + s["bias"].double()
    out = [y, stream] if case["residual"] else [y]
    if case["kind"] == "norm":
        return tuple(out) if case["residual"] else y
    dy = s["grads"][0].double()
    # y depends on x_j by way of itself, the mean and the variance.
    d_centred = dy * w / root
    d_variance = -0.5 * (dy * w * (x - mean)).sum(-1, keepdim=True) / root ** 3
    dx = d_centred - d_centred.mean(-1, keepdim=True) + 2.0 / case["dim"] * d_variance * (x - mean)
    if case["residual"]:
        dx += s["grads"][1].double()
    out += [dx, (dy * (x - mean) / root).sum(0), dy.sum(0)]
    return tuple(out + ([dx] if case["residual"] else []))


def _exact_linear(case, s):
    """Token by token, and back token by token."""
    share = case["value_heads"] // case["key_heads"]
    q, k, v, g, state = (s[n].detach().double() for n in ("q", "k", "v", "g", "state"))
    q, k = q.repeat_interleave(share, 2), k.repeat_interleave(share, 2)
    decay = g.exp().expand(v.shape[:3])
    if s["reset"] is not None:
        decay = torch.where(s["reset"][..., None], torch.zeros_like(decay), decay)
    decay = decay[..., None, None]
    o, states = torch.empty_like(v), [state]
    for t in range(case["length"]):
        state = decay[:, t] * state + k[:, t, :, :, None] * v[:, t, :, None, :]
        o[:, t] = s["scale"] * (state * q[:, t, :, :, None]).sum(-2)
        if case["kind"] == "train":
            states.append(state)
    if case["kind"] == "step":
        return o[:, 0], state
    if case["kind"] == "forward":
        return o, state
    do, ds = s["grads"][0].double(), s["grads"][1].double()
    dq, dk, dv, dg = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v), torch.zeros_like(g)
    for t in reversed(range(case["length"])):
        out = s["scale"] * do[:, t, :, None, :]
        dq[:, t] = (states.pop() * out).sum(-1)
        ds = ds + q[:, t, :, :, None] * out
        dk[:, t] = (ds * v[:, t, :, None, :]).sum(-1)
        dv[:, t] = (ds * k[:, t, :, :, None]).sum(-2)
        ds = decay[:, t] * ds
        if case["learned"]:
            dg += (ds * states[-1]).sum((0, 2, 3))
    dq, dk = (x.unflatten(2, (-1, share)).sum(3) for x in (dq, dk))
    return (o, state, dq, dk, dv, ds) + ((dg,) if case["learned"] else ())
