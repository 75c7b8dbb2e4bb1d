"""Cases for the policy operators: the gated delta rule over a rollout (forward, and with its gradients),
its one-token form that acts in every environment, and the Newton-Schulz orthogonalisation of an update.

Each case names an operator and its sizes.  ``run`` computes one pass, either in a plain form (elementary
32-bit torch operations) or, where ``own`` is true, through the package's entry points."""
import math

import torch

own = False

NS_COEFFICIENTS = (3.4445, -4.7750, 2.0315)
NORM_EPS = 1e-6  # under the root of the per-head norms of q and k
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def _delta(name, op, batch, tokens, heads, key_heads, dk, dv, dtype, reset, state, time_major=False):
    return {"name": name, "op": op, "batch": batch, "tokens": tokens, "heads": heads, "key_heads": key_heads, "dk": dk,
            "dv": dv, "dtype": dtype, "reset": reset, "state": state, "time_major": time_major}


def _orth(name, count, rows, cols, dtype):
    return {"name": name, "op": "orthogonalize", "count": count, "rows": rows, "cols": cols, "dtype": dtype}


def listed():
    return [
        # acting in one environment (evaluation, a viewer): the smallest call, latency alone
        _delta("step one env", "step", 1, 1, 4, 4, 64, 64, "bf16", 0.0, True),
        # acting in the benchmark's 16384 environments, episodes of about 1000 steps
        _delta("step 16384 envs", "step", 16384, 1, 4, 4, 64, 64, "bf16", 0.001, True),
        # 32-bit policy, odd head sizes, one key head shared by three value heads, frequent episode ends
        _delta("step odd f32", "step", 777, 1, 3, 1, 40, 56, "f32", 0.1, True),
        # values of a rollout of 4096 environments (bootstrapping, old log-probabilities): no gradients
        _delta("rollout 4096x32", "forward", 4096, 32, 4, 4, 64, 64, "bf16", 0.01, True, True),
        # few long recorded episodes: no parallelism in the batch
        _delta("long 2x4096", "forward", 2, 4096, 8, 4, 128, 128, "bf16", 0.001, False),
        # 32-bit, ragged: an odd number of tokens, environments and channels
        _delta("ragged forward f32", "forward", 61, 101, 3, 1, 40, 56, "f32", 0.02, True),
        # the learning step of a rollout: outputs and all gradients, time-major storage as a rollout buffer has it
        _delta("train 4096x32", "train", 4096, 32, 4, 4, 64, 64, "bf16", 0.01, False, True),
        # whole episodes of 1000 steps, few of them, wide shared heads, a learned initial state
        _delta("train 8x1000", "train", 8, 1000, 8, 4, 128, 128, "bf16", 0.001, True),
        # 32-bit learning step with odd sizes throughout
        _delta("train ragged f32", "train", 173, 77, 3, 3, 40, 24, "f32", 0.02, True),
        # the first layer of a small policy: 29 observations to 64 units
        _orth("orth 64x29", 1, 64, 29, "f32"),
        # the stacked projections of a policy's layers, 16-bit
        _orth("orth 8x512x1024", 8, 512, 1024, "bf16"),
        # a large matrix in 32 bits
        _orth("orth 2048x2048", 1, 2048, 2048, "f32"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["step", "forward", "train", "orthogonalize"])
    dtype = rng.choice(["bf16", "f32"])
    if op == "orthogonalize":
        while True:
            rows, cols, count = _log_int(rng, 16, 2048), _log_int(rng, 16, 2048), _log_int(rng, 1, 16)
            if count * rows * cols * min(rows, cols) <= 2048 ** 3:
                break
        c = _orth("", count, rows, cols, dtype)
    else:
        key_heads = rng.choice([1, 2, 3, 4])
        heads = key_heads * rng.choice([1, 1, 2])
        dk, dv = rng.choice([64, 128, 8 * rng.randint(2, 16)]), rng.choice([64, 128, 8 * rng.randint(2, 16)])
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
        c = _delta("", op, batch, tokens, heads, key_heads, dk, dv, dtype, reset, rng.random() < 0.5 or op == "step",
                   rng.random() < 0.5)
    del c["name"]
    return c


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device=dev)

    dtype = DTYPES[case["dtype"]]
    if case["op"] == "orthogonalize":
        n, r, c = case["count"], case["rows"], case["cols"]
        # a momentum buffer: a strong low-rank part (the gradient's main directions) over noise
        rank = max(1, min(r, c) // 8)
        m = normal(n, r, c) + normal(n, r, rank) @ normal(n, rank, c) / math.sqrt(rank)
        return {"op": "orthogonalize", "update": (0.01 * m).to(dtype)}
    B, T, H, K, dk, dv = (case[x] for x in ("batch", "tokens", "heads", "key_heads", "dk", "dv"))

    def rollout(x):  # [B, T, ...] as seen by the operator, stored [T, B, ...] where the buffer is time-major
        return x.transpose(0, 1).contiguous().transpose(0, 1) if case["time_major"] else x

    q, k, v = normal(B, T, K, dk), normal(B, T, K, dk), normal(B, T, H, dv)
    # decays of a gate: exp(g) from 0.6 to nearly 1; write strengths of a sigmoid
    g = -torch.rand((B, T, H), generator=gen, device=dev).square() * 0.5
    beta = torch.sigmoid(normal(B, T, H))
    reset = (torch.rand((B, T), generator=gen, device=dev) < case["reset"]).to(torch.uint8)
    state = {"op": case["op"], "q": rollout(q.to(dtype)), "k": rollout(k.to(dtype)), "v": rollout(v.to(dtype)),
             "g": rollout(g), "beta": rollout(beta), "reset": rollout(reset) if case["reset"] else None,
             "initial": 0.3 * normal(B, H, dk, dv) if case["state"] else None}
    if case["op"] == "step":
        for x in ("q", "k", "v", "g", "beta", "reset"):
            state[x] = state[x][:, 0].contiguous() if state[x] is not None else None
    if case["op"] == "train":
        state["d_out"] = rollout(normal(B, T, H, dv).to(dtype))
        for x in ("q", "k", "v", "g", "beta", "initial"):
            if state[x] is not None:
                state[x].requires_grad_(True)
    return state


def _heads(x, heads):
    """Key heads repeated for the value heads that share them; [B, T, H, d] to [B, H, T, d] in 32 bits."""
    return x.float().repeat_interleave(heads // x.shape[2], dim=2).transpose(1, 2)


def _unit_lower_inverse(n):
    """(I + n)^-1 of strictly lower triangular n by doubling the block size."""
    size = n.shape[-1]
    inv = torch.eye(size, device=n.device).expand_as(n)
    at = torch.arange(size, device=n.device)
    block = 1
    while block < size:
        # the lower left quarters of the diagonal blocks twice as large
        low = (at[:, None] // block % 2 == 1) & (at[None, :] // block == at[:, None] // block - 1)
        inv = inv - inv @ (n * low) @ inv
        block *= 2
    return inv


def _plain_delta(q, k, v, g, beta, reset, initial):
    """The chunked form in 32-bit torch operations: ([B, T, H, dv] 32-bit outputs, final state)."""
    B, T, H, dv = v.shape
    dk, chunk = q.shape[-1], min(64, T)
    pad = -T % chunk
    q, k, v = (torch.nn.functional.pad(_heads(x, H), (0, 0, 0, pad)) for x in (q, k, v))
    q = q * (q.square().sum(-1, keepdim=True) + NORM_EPS).rsqrt() * dk ** -0.5
    k = k * (k.square().sum(-1, keepdim=True) + NORM_EPS).rsqrt()
    g, beta = (torch.nn.functional.pad(x.transpose(1, 2), (0, pad)) for x in (g, beta))
    r = torch.zeros((B, 1, T + pad), device=q.device, dtype=torch.bool)
    if reset is not None:
        r[:, 0, :T] = reset != 0
    n = (T + pad) // chunk
    q, k, v = (x.reshape(B, H, n, chunk, -1) for x in (q, k, v))
    g, beta, r = (x.reshape(B, -1, n, chunk) for x in (g, beta, r))
    episode = r.long().cumsum(-1)
    total = torch.where(r, torch.zeros_like(g), g).cumsum(-1)
    same = (episode[..., :, None] == episode[..., None, :]).tril()
    decay = torch.where(same, total[..., :, None] - total[..., None, :], torch.full((), -math.inf, device=q.device)).exp()
    carried = torch.where(episode == 0, total, torch.full((), -math.inf, device=q.device)).exp()
    inverse = _unit_lower_inverse((k @ k.mT * decay * beta[..., None, :]).tril(-1))
    scores = q @ k.mT * decay
    state = initial if initial is not None else torch.zeros((B, H, dk, dv), device=q.device)
    out = []
    for c in range(n):
        a = carried[:, :, c, :, None]
        u = beta[:, :, c, :, None] * (inverse[:, :, c] @ (v[:, :, c] - a * (k[:, :, c] @ state)))
        out.append(a * (q[:, :, c] @ state) + scores[:, :, c] @ u)
        state = a[:, :, -1:] * state + k[:, :, c].mT @ (decay[:, :, c, -1, :, None] * u)
    return torch.cat(out, 2)[:, :, :T].transpose(1, 2), state


def _plain_step(s):
    H, dk = s["v"].shape[1], s["q"].shape[-1]
    q, k = (x.float().repeat_interleave(H // x.shape[1], dim=1) for x in (s["q"], s["k"]))
    q = q * (q.square().sum(-1, keepdim=True) + NORM_EPS).rsqrt() * dk ** -0.5
    k = k * (k.square().sum(-1, keepdim=True) + NORM_EPS).rsqrt()
    alpha = s["g"].exp()
    if s["reset"] is not None:
        alpha = alpha * (s["reset"] == 0)[:, None]
    state = s["initial"]
    state.mul_(alpha[..., None, None])
    u = s["beta"][..., None] * (s["v"].float() - (k[..., None, :] @ state)[..., 0, :])
    state.add_(k[..., None] * u[..., None, :])
    return {"out": (q[..., None, :] @ state)[..., 0, :].to(s["v"].dtype), "state": state}


def _plain_orthogonalize(update):
    x = update.float()
    x = x.mT if x.shape[-2] > x.shape[-1] else x
    x = x / (x.square().sum((-2, -1), keepdim=True).sqrt() + 1e-7)
    a, b, c = NS_COEFFICIENTS
    for _ in range(5):
        gram = x @ x.mT
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    x = x.mT if update.shape[-2] > update.shape[-1] else x
    return x.to(update.dtype).contiguous()


def run(s):
    if s["op"] == "orthogonalize":
        if own:
            import zeno_b200
            return zeno_b200.orthogonalize(s["update"])
        return _plain_orthogonalize(s["update"])
    if s["op"] == "step":
        if own:
            import zeno_b200
            out = zeno_b200.delta_rule_step(s["q"], s["k"], s["v"], s["g"], s["beta"], s["initial"], s["reset"])
            return {"out": out, "state": s["initial"]}
        return _plain_step(s)
    args = [s[x] for x in ("q", "k", "v", "g", "beta", "reset", "initial")]
    with torch.set_grad_enabled(s["op"] == "train"):
        if own:
            import zeno_b200
            out, final = zeno_b200.delta_rule(*args)
        else:
            out, final = _plain_delta(*args)
            out = out.to(s["v"].dtype)
    got = {"out": out, "state": final}
    if s["op"] == "train":
        names = [x for x in ("q", "k", "v", "g", "beta", "initial") if s[x] is not None]
        for x, grad in zip(names, torch.autograd.grad(out, [s[x] for x in names], s["d_out"])):
            got["d_" + x] = grad
    return got


def work(case):
    size = DTYPES[case["dtype"]].itemsize
    if case["op"] == "orthogonalize":
        n, m, k = case["count"], min(case["rows"], case["cols"]), max(case["rows"], case["cols"])
        # the two symmetric products need half their entries
        return {"bytes": 2 * n * m * k * size, "flops": 5 * n * (m * (m + 1) * k + m * (m + 1) * m + 2 * m * m * k)}
    B, T, H, K, dk, dv = (case[x] for x in ("batch", "tokens", "heads", "key_heads", "dk", "dv"))
    vectors = B * T * (2 * K * dk + 2 * H * dv) * size + B * T * H * 8 + (B * T if case["reset"] else 0)
    states = B * H * dk * dv * 4 * (2 if case["state"] else 1)
    flops = 6 * B * T * H * dk * dv
    if case["op"] == "train":  # also reads the outputs' gradient, writes those of q, k, v, the gates and the first state
        vectors += B * T * (2 * K * dk + 2 * H * dv) * size + B * T * H * 8
        states += B * H * dk * dv * 4 if case["state"] else 0
        flops *= 3
    return {"bytes": vectors + states, "flops": flops}


def _exact_delta(s, part):
    """One slice of the batch, token by token in 64 bits; the gradients by the reverse recurrence."""
    v = s["v"].detach()[part].double()
    H, dk = v.shape[2], s["q"].shape[-1]
    group = H // s["q"].shape[2]
    raw_q, raw_k, v = (s[x].detach()[part].double() for x in ("q", "k", "v"))
    norm_q = (raw_q.pow(2).sum(-1, keepdim=True) + NORM_EPS).sqrt()
    norm_k = (raw_k.pow(2).sum(-1, keepdim=True) + NORM_EPS).sqrt()
    hat_q, hat_k = raw_q / norm_q, raw_k / norm_k
    q, k = (x.repeat_interleave(group, 2) for x in (hat_q * dk ** -0.5, hat_k))
    alpha = s["g"].detach()[part].double().exp()
    beta = s["beta"].detach()[part].double()
    if s["reset"] is not None:
        alpha = alpha * (s["reset"][part] == 0).double()[..., None]
    S = s["initial"].detach()[part].double() if s["initial"] is not None else v.new_zeros((v.shape[0], H, dk, v.shape[-1]))
    train = s["op"] == "train"
    out, before, errors = torch.empty_like(v), [], []
    for t in range(v.shape[1]):
        if train:
            before.append(S)
        decayed = alpha[:, t, :, None, None] * S
        error = v[:, t] - torch.einsum("bhkv,bhk->bhv", decayed, k[:, t])
        S = decayed + torch.einsum("bhk,bhv->bhkv", k[:, t], beta[:, t, :, None] * error)
        out[:, t] = torch.einsum("bhkv,bhk->bhv", S, q[:, t])
        errors.append(error if train else None)
    got = {"out": out, "state": S}
    if not train:
        return got
    d_out = s["d_out"][part].double()
    d_q, d_k, d_v, d_g, d_beta = (torch.empty_like(x) for x in (q, k, v, alpha, beta))
    R = torch.zeros_like(S)
    for t in reversed(range(v.shape[1])):
        decayed = alpha[:, t, :, None, None] * before[t]
        u = beta[:, t, :, None] * errors[t]
        after = decayed + torch.einsum("bhk,bhv->bhkv", k[:, t], u)
        d_q[:, t] = torch.einsum("bhkv,bhv->bhk", after, d_out[:, t])
        R = R + torch.einsum("bhk,bhv->bhkv", q[:, t], d_out[:, t])
        d_u = torch.einsum("bhkv,bhk->bhv", R, k[:, t])
        d_beta[:, t] = (d_u * errors[t]).sum(-1)
        d_v[:, t] = beta[:, t, :, None] * d_u
        d_k[:, t] = torch.einsum("bhkv,bhv->bhk", R, u) - torch.einsum("bhkv,bhv->bhk", decayed, d_v[:, t])
        R = R - torch.einsum("bhk,bhv->bhkv", k[:, t], d_v[:, t])
        d_g[:, t] = (R * decayed).sum((-2, -1))
        R = alpha[:, t, :, None, None] * R

    def shared(d, hat, norm):  # the sum over the heads that share a key head, then back through the norm
        d = d.unflatten(2, (-1, group)).sum(3)
        return (d - hat * (hat * d).sum(-1, keepdim=True)) / norm

    got.update(d_q=shared(d_q * dk ** -0.5, hat_q, norm_q), d_k=shared(d_k, hat_k, norm_k), d_v=d_v, d_g=d_g, d_beta=d_beta)
    if s["initial"] is not None:
        got["d_initial"] = R
    return got


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "orthogonalize":
        m = s["update"].double()
        wide = m.shape[-2] <= m.shape[-1]
        x = (m if wide else m.transpose(-2, -1)) / (torch.linalg.matrix_norm(m)[..., None, None] + 1e-7)
        a, b, c = NS_COEFFICIENTS
        for _ in range(5):  # a x + b (x x') x + c (x x')^2 x, from the right
            once = torch.bmm(torch.bmm(x, x.transpose(1, 2)), x)
            x = a * x + b * once + c * torch.bmm(torch.bmm(x, x.transpose(1, 2)), once)
        return x if wide else x.transpose(-2, -1).contiguous()
    if case["op"] == "step":
        for x in ("q", "k", "v", "g", "beta", "reset"):
            s[x] = s[x][:, None] if s[x] is not None else None
    # slices of the batch that hold about 4 GB of states
    per = case["tokens"] * case["heads"] * case["dk"] * case["dv"] * 8
    size = max(1, int(4e9 // per)) if case["op"] == "train" else max(1, int(4e9 // (per / case["tokens"])))
    parts = [_exact_delta(s, slice(i, i + size)) for i in range(0, case["batch"], size)]
    got = {x: torch.cat([p[x] for p in parts]) for x in parts[0]}
    if case["op"] == "step":
        got["out"] = got["out"][:, 0]
    return got
