"""Cases for the memory with a decay for each head (linear attention over a rollout, forward and with its gradients, and
its one-token form that acts in every environment) and for layer norm (forward, and with its gradients).

Each case names an operator and its sizes.  ``run`` computes one pass, either in a plain form (elementary
32-bit torch operations) or, where ``own`` is true, through the package's entry points."""
import math

import torch

own = False

NORM_EPS = 1e-5
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def _attention(name, op, batch, tokens, heads, key_heads, dk, dv, dtype, reset, state, fixed, time_major=False):
    return {"name": name, "op": op, "batch": batch, "tokens": tokens, "heads": heads, "key_heads": key_heads, "dk": dk,
            "dv": dv, "dtype": dtype, "reset": reset, "state": state, "fixed": fixed, "time_major": time_major}


def _norm(name, op, rows, width, dtype, affine):
    return {"name": name, "op": op, "rows": rows, "width": width, "dtype": dtype, "affine": affine}


def listed():
    return [
        # acting in one environment (evaluation, a viewer): the smallest call, latency alone
        _attention("step one env", "step", 1, 1, 4, 4, 64, 64, "bf16", 0.0, True, True),
        # acting in the benchmark's 16384 environments, episodes of about 1000 steps, one decay for each head
        _attention("step 16384 envs", "step", 16384, 1, 4, 4, 64, 64, "bf16", 0.001, True, True),
        # 32-bit policy, odd head sizes, one key head shared by three value heads, gated decays, frequent episode ends
        _attention("step odd f32", "step", 777, 1, 3, 1, 40, 56, "f32", 0.1, True, False),
        # values of a rollout of 4096 environments (bootstrapping, old log-probabilities): no gradients
        _attention("rollout 4096x32", "forward", 4096, 32, 4, 4, 64, 64, "bf16", 0.01, True, True, True),
        # few long recorded episodes: no parallelism in the batch
        _attention("long 2x4096", "forward", 2, 4096, 8, 4, 128, 128, "bf16", 0.001, False, True),
        # the learning step of a rollout: outputs and all gradients, time-major storage as a rollout buffer has it
        _attention("train 4096x32", "train", 4096, 32, 4, 4, 64, 64, "bf16", 0.01, False, True, True),
        # whole episodes of 1000 steps, few of them, wide shared heads, gated decays, a learned initial state
        _attention("train 8x1000", "train", 8, 1000, 8, 4, 128, 128, "bf16", 0.001, True, False),
        # 32-bit learning step with odd sizes throughout
        _attention("train ragged f32", "train", 173, 77, 3, 3, 40, 24, "f32", 0.02, True, False),
        # the features of one environment in front of a policy's projections: latency alone
        _norm("norm one env", "norm", 1, 256, "f32", True),
        # what a memory of 4 heads returns for a rollout of 4096 x 32, each head's 64 channels on their own
        _norm("norm reads", "norm", 524288, 64, "bf16", False),
        # the hidden layer of the same rollout, with gradients of input, weight and bias
        _norm("norm train 131072x256", "norm_train", 131072, 256, "bf16", True),
        # a wide 32-bit layer of an odd width, few rows
        _norm("norm train odd f32", "norm_train", 2047, 4099, "f32", True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["step", "forward", "train", "norm", "norm_train"])
    dtype = rng.choice(["bf16", "f32"])
    if op in ("norm", "norm_train"):
        width = _log_int(rng, 16, 8192)
        c = _norm("", op, _log_int(rng, 1, 131072 * 256 // 2 // width), width, dtype, rng.random() < 0.7)
    else:
        key_heads = rng.choice([1, 2, 3, 4])
        heads = key_heads * rng.choice([1, 1, 2])
        dk, dv = rng.choice([64, 128, 8 * rng.randint(2, 16), rng.randint(9, 99)]), rng.choice([64, 128, 8 * rng.randint(2, 16), rng.randint(9, 99)])
        reset = rng.choice([0.0, 0.001, 0.02, 0.1])
        if op == "step":
            most = 16384 * 4 * 64 * 64
            batch, tokens = min(_log_int(rng, 1, 16384), most // (heads * dk * dv)), 1
        else:
            # as many token-heads as the listed rollout has, weighed by the head's size
            most = 4096 * 32 * 4 * 64 * 64 // (heads * dk * dv)
            tokens = _log_int(rng, 2, 4096)
            batch = max(1, min(_log_int(rng, 1, 4096), most // tokens))
            if tokens > 1024 and op == "train":
                tokens = rng.randint(100, 1024)
        c = _attention("", op, batch, tokens, heads, key_heads, dk, dv, dtype, reset, rng.random() < 0.5 or op == "step",
                       rng.random() < 0.5, rng.random() < 0.5)
    del c["name"]
    return c


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device=dev)

    def uniform(*shape):
        return torch.rand(shape, generator=gen, device=dev)

    dtype = DTYPES[case["dtype"]]
    if case["op"] in ("norm", "norm_train"):
        n, d = case["rows"], case["width"]
        # activations of channels with their own means and spreads, rows of different sizes
        x = (normal(n, d) * (0.5 + uniform(d)) + 0.5 * normal(d)) * torch.exp(normal(n, 1))
        state = {"op": case["op"], "x": x.to(dtype), "weight": None, "bias": None}
        if case["affine"]:
            state["weight"], state["bias"] = 1 + 0.1 * normal(d), 0.1 * normal(d)
        if case["op"] == "norm_train":
            state["d_out"] = normal(n, d).to(dtype)
            for name in ("x", "weight", "bias"):
                if state[name] is not None:
                    state[name].requires_grad_(True)
        return state
    B, T, H, K, dk, dv = (case[x] for x in ("batch", "tokens", "heads", "key_heads", "dk", "dv"))

    def rollout(x):  # [B, T, ...] as seen by the operator, stored [T, B, ...] where the buffer is time-major
        return x.transpose(0, 1).contiguous().transpose(0, 1) if case["time_major"] else x

    q, k, v = normal(B, T, K, dk), normal(B, T, K, dk) * dk ** -0.25, normal(B, T, H, dv)
    if case["fixed"]:
        # one learned log decay for each head, memories of about 4 to 256 tokens
        g = -(2.0 ** (-2 - 6 * uniform(H)))
    else:
        # decays of a gate: exp(g) from 0.6 to nearly 1
        g = rollout(-uniform(B, T, H).square() * 0.5)
    reset = (uniform(B, T) < case["reset"]).to(torch.uint8)
    state = {"op": case["op"], "q": rollout(q.to(dtype)), "k": rollout(k.to(dtype)), "v": rollout(v.to(dtype)), "g": g,
             "reset": rollout(reset) if case["reset"] else None, "initial": 0.3 * normal(B, H, dk, dv) if case["state"] else None}
    if case["op"] == "step":
        for x in ("q", "k", "v", "g", "reset"):
            if state[x] is not None and not (x == "g" and case["fixed"]):
                state[x] = state[x][:, 0].contiguous()
    if case["op"] == "train":
        state["d_out"] = rollout(normal(B, T, H, dv).to(dtype))
        # where a memory is handed in it is handed on, and the loss reaches back through it
        state["d_last"] = 0.3 * normal(B, H, dk, dv) if case["state"] else None
        for x in ("q", "k", "v", "g", "initial"):
            if state[x] is not None:
                state[x].requires_grad_(True)
    return state


def _plain_attention(q, k, v, g, reset, initial):
    """The chunked form in 32-bit torch operations (sums of log decays in 64): (outputs [B, T, H, dv], final state)."""
    B, T, H, dv = v.shape
    dk, chunk = q.shape[-1], min(64, T)
    pad, n = -T % chunk, -(-T // chunk)
    # [B, T, heads, width] to [B, H, chunks, chunk, width]
    q, k, v = (torch.nn.functional.pad(x.float().repeat_interleave(H // x.shape[2], dim=2).transpose(1, 2), (0, 0, 0, pad))
               .reshape(B, H, n, chunk, -1) for x in (q, k, v))
    g = torch.nn.functional.pad(g.double().expand(B, T, H).transpose(1, 2), (0, pad))
    r = torch.zeros((B, 1, T + pad), device=q.device, dtype=torch.bool)
    if reset is not None:
        r[:, 0, :T] = reset != 0
    total = torch.where(r, torch.zeros_like(g), g).cumsum(-1).reshape(B, H, n, chunk)
    episode = r.long().cumsum(-1).reshape(B, 1, n, chunk)

    def decay(mask, log):
        return torch.where(mask, log, torch.full((), -math.inf, dtype=log.dtype, device=log.device)).float().exp()

    same = (episode[..., :, None] == episode[..., None, :]).tril()
    scores = q @ k.mT * decay(same, total[..., :, None] - total[..., None, :])
    # what each chunk adds to the state at its end, and the states in front of the chunks from those before
    last, last_episode = total[..., -1], episode[..., -1]
    added = (k * decay(episode == last_episode[..., None], last[..., None] - total)[..., None]).mT @ v
    before = torch.nn.functional.pad(last, (1, 0))  # sums and episodes in front of chunk 0, 1, ..., n
    before_episode = torch.nn.functional.pad(last_episode, (1, 0))
    reach = torch.ones((n + 1, n), dtype=torch.bool, device=q.device).tril(-1)
    onward = decay(reach & (before_episode[..., :, None] == last_episode[..., None, :]), before[..., :, None] - last[..., None, :])
    states = torch.einsum("bhcj,bhjkv->bhckv", onward, added)
    if initial is not None:
        states = states + decay(before_episode == 0, before)[..., None, None] * initial[:, :, None]
    carried = decay(episode == before_episode[..., :-1, None], total - before[..., :-1, None])
    out = scores @ v + carried[..., None] * (q @ states[:, :, :-1])
    return (out * dk ** -0.5).reshape(B, H, T + pad, dv)[:, :, :T].transpose(1, 2), states[:, :, -1]


def _plain_step(s):
    H, dk = s["v"].shape[1], s["q"].shape[-1]
    q, k = (x.float().repeat_interleave(H // x.shape[1], dim=1) for x in (s["q"], s["k"]))
    alpha = s["g"].exp().expand(q.shape[0], H)
    if s["reset"] is not None:
        alpha = alpha * (s["reset"] == 0)[:, None]
    state = s["initial"]
    state.mul_(alpha[..., None, None])
    state.add_(k[..., None] * s["v"].float()[..., None, :])
    return {"out": ((q[..., None, :] @ state)[..., 0, :] * dk ** -0.5).to(s["v"].dtype), "state": state}


def _plain_norm(x, weight, bias):
    y = x.float()
    y = y - y.mean(-1, keepdim=True)
    y = y * (y.square().mean(-1, keepdim=True) + NORM_EPS).rsqrt()
    if weight is not None:
        y = y * weight + bias
    return y.to(x.dtype)


def _gradients(s, names, outputs, seeds):
    names = [x for x in names if s[x] is not None]
    return {"d_" + x: grad for x, grad in zip(names, torch.autograd.grad(outputs, [s[x] for x in names], seeds))}


def run(s):
    if s["op"] in ("norm", "norm_train"):
        with torch.set_grad_enabled(s["op"] == "norm_train"):
            if own:
                import zeno_b200
                out = zeno_b200.layer_norm(s["x"], s["weight"], s["bias"], eps=NORM_EPS)
            else:
                out = _plain_norm(s["x"], s["weight"], s["bias"])
        got = {"out": out}
        if s["op"] == "norm_train":
            got.update(_gradients(s, ("x", "weight", "bias"), [out], [s["d_out"]]))
        return got
    if s["op"] == "step":
        if own:
            import zeno_b200
            out = zeno_b200.linear_attention_step(s["q"], s["k"], s["v"], s["g"], s["initial"], s["reset"])
            return {"out": out, "state": s["initial"]}
        return _plain_step(s)
    args = [s[x] for x in ("q", "k", "v", "g", "reset", "initial")]
    with torch.set_grad_enabled(s["op"] == "train"):
        if own:
            import zeno_b200
            out, final = zeno_b200.linear_attention(*args)
        else:
            out, final = _plain_attention(*args)
            out = out.to(s["v"].dtype)
    got = {"out": out, "state": final}
    if s["op"] == "train":
        outputs, seeds = [out], [s["d_out"]]
        if s["d_last"] is not None:
            outputs, seeds = [out, final], [s["d_out"], s["d_last"]]
        got.update(_gradients(s, ("q", "k", "v", "g", "initial"), outputs, seeds))
    return got


def work(case):
    size = DTYPES[case["dtype"]].itemsize
    if case["op"] in ("norm", "norm_train"):
        n, d = case["rows"], case["width"]
        train = case["op"] == "norm_train"  # also reads the outputs' gradient, writes those of x, weight and bias
        return {"bytes": n * d * size * (4 if train else 2) + (d * 4 * (4 if train else 2) if case["affine"] else 0),
                "flops": n * d * (20 if train else 8)}
    B, T, H, K, dk, dv = (case[x] for x in ("batch", "tokens", "heads", "key_heads", "dk", "dv"))
    gates = H if case["fixed"] else B * T * H
    vectors = B * T * (2 * K * dk + 2 * H * dv) * size + gates * 4 + (B * T if case["reset"] else 0)
    states = B * H * dk * dv * 4 * (2 if case["state"] else 1)
    flops = 4 * B * T * H * dk * dv
    if case["op"] == "train":  # also reads the outputs' gradients, writes those of q, k, v, the gates and the first state
        vectors += B * T * (2 * K * dk + 2 * H * dv) * size + gates * 4
        states *= 2 if case["state"] else 1
        flops *= 3
    return {"bytes": vectors + states, "flops": flops}


def _exact_attention(s, part):
    """One slice of the batch, token by token in 64 bits; the gradients by the reverse recurrence."""
    raw_q, raw_k, v = (s[x].detach()[part].double() for x in ("q", "k", "v"))
    B, T, H, dv = v.shape
    dk, group = raw_q.shape[-1], H // raw_q.shape[2]
    q, k = raw_q.repeat_interleave(group, 2) * dk ** -0.5, raw_k.repeat_interleave(group, 2)
    g = s["g"].detach().double()
    alpha = (g.expand(B, T, H) if g.dim() == 1 else g[part]).exp()
    if s["reset"] is not None:
        alpha = alpha * (s["reset"][part] == 0).double()[..., None]
    S = s["initial"].detach()[part].double() if s["initial"] is not None else v.new_zeros((B, H, dk, dv))
    train = s["op"] == "train"
    out, before = torch.empty_like(v), []
    for t in range(T):
        if train:
            before.append(S)
        S = alpha[:, t, :, None, None] * S + torch.einsum("bhk,bhv->bhkv", k[:, t], v[:, t])
        out[:, t] = torch.einsum("bhkv,bhk->bhv", S, q[:, t])
    got = {"out": out, "state": S}
    if not train:
        return got
    d_out = s["d_out"][part].double()
    d_q, d_k, d_v, d_g = (torch.empty_like(x) for x in (q, k, v, alpha))
    R = s["d_last"][part].double() if s["d_last"] is not None else torch.zeros_like(S)
    for t in reversed(range(T)):
        decayed = alpha[:, t, :, None, None] * before[t]
        after = decayed + torch.einsum("bhk,bhv->bhkv", k[:, t], v[:, t])
        d_q[:, t] = torch.einsum("bhkv,bhv->bhk", after, d_out[:, t]) * dk ** -0.5
        R = R + torch.einsum("bhk,bhv->bhkv", q[:, t], d_out[:, t])
        d_k[:, t] = torch.einsum("bhkv,bhv->bhk", R, v[:, t])
        d_v[:, t] = torch.einsum("bhkv,bhk->bhv", R, k[:, t])
        d_g[:, t] = (R * decayed).sum((-2, -1))
        R = alpha[:, t, :, None, None] * R
    # the sums over the value heads that share a key head
    got.update(d_q=d_q.unflatten(2, (-1, group)).sum(3), d_k=d_k.unflatten(2, (-1, group)).sum(3), d_v=d_v, d_g=d_g)
    if s["initial"] is not None:
        got["d_initial"] = R
    return got


def _exact_norm(s):
    x = s["x"].detach().double()
    d = x.shape[-1]
    var, mean = torch.var_mean(x, -1, correction=0, keepdim=True)
    std = (var + NORM_EPS).sqrt()
    hat = (x - mean) / std
    affine = s["weight"] is not None
    w = s["weight"].detach().double() if affine else torch.ones(d, dtype=torch.float64, device=x.device)
    got = {"out": torch.addcmul(s["bias"].detach().double(), hat, w) if affine else hat}
    if s["op"] == "norm_train":
        dy = s["d_out"].double()
        dh = dy * w
        got["d_x"] = (dh - dh.sum(-1, keepdim=True) / d - hat * ((dh * hat).sum(-1, keepdim=True) / d)) / std
        if affine:
            got["d_weight"], got["d_bias"] = (dy * hat).sum(0), dy.sum(0)
    return got


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("norm", "norm_train"):
        return _exact_norm(s)
    if case["op"] == "step":
        for x in ("q", "k", "v", "reset"):
            s[x] = s[x][:, None] if s[x] is not None else None
        s["g"] = s["g"] if case["fixed"] else s["g"][:, None]
    # slices of the batch that hold about 4 GB of states
    per = case["tokens"] * case["heads"] * case["dk"] * case["dv"] * 8
    size = max(1, int(4e9 // per)) if case["op"] == "train" else max(1, int(4e9 // (per / case["tokens"])))
    parts = [_exact_attention(s, slice(i, i + size)) for i in range(0, case["batch"], size)]
    got = {x: torch.cat([p[x] for p in parts]) for x in parts[0]}
    if case["op"] == "step":
        got["out"] = got["out"][:, 0]
    if case["op"] == "train" and case["fixed"]:
        got["d_g"] = got["d_g"].sum((0, 1))
    return got
