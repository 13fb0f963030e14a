"""Operators of policies that are trained as low-rank adapters of one shared
model, as they are measured: the calls of a user's program, their inputs, their
plain form in elementary torch operations, what each cannot do without, and
their 64-bit results.

* ``sample``: a token a row from given uniforms, every row with its own
  temperature, top-k, top-p and min-p (``rosellm_amd.roseinfer.sample_tokens``).
* ``adapters`` / ``adapters_step``: the low-rank updates of many requests'
  adapters beside a shared projection, and with their gradients
  (``rosellm_amd.rosetrainer.adapter_linear``).
* ``dropout`` / ``dropout_step``: dropout whose mask is drawn again instead of
  stored, and with its gradient (``rosellm_amd.rosetrainer.dropout``).
"""

import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_SIZES = {"bf16": 2, "f16": 2, "f32": 4}

# Consecutive entries of a row that one call of the generator serves, 16 bits each.
_GROUP = 8


def listed():
    return [
        # one sequence of a low-latency rollout
        dict(name="sample_one", op="sample", B=1, V=151936, dtype="bf16", settings="nucleus"),
        # a rollout batch that is drawn from the policy itself
        dict(name="sample_policy", op="sample", B=64, V=151936, dtype="bf16", settings="none"),
        # a full batch of requests, each with settings of its own, some greedy
        dict(name="sample_mixed", op="sample", B=256, V=151936, dtype="bf16", settings="mixed"),
        # float32 logits of an odd vocabulary
        dict(name="sample_odd_f32", op="sample", B=37, V=50257, dtype="f32", settings="top_k"),
        # one decode step: every request has its own adapter, or none
        dict(name="adapters_decode", op="adapters", N=64, A=16, H=1024, O=2048, r=16, dtype="bf16", runs=1),
        # the same step's adapters of the LM head
        dict(name="adapters_head", op="adapters", N=16, A=8, H=1024, O=151936, r=16, dtype="bf16", runs=1),
        # prompts of several requests in one batch
        dict(name="adapters_prompts", op="adapters", N=8192, A=8, H=1024, O=4096, r=32, dtype="bf16", runs=700),
        # the training step of one policy, 128 x 1024 tokens
        dict(name="adapters_step", op="adapters_step", N=131072, A=1, H=1024, O=2048, r=16, dtype="bf16", runs=131072, p=0.05),
        # a short float32 step of three policies, odd sizes
        dict(name="adapters_step_odd", op="adapters_step", N=1000, A=3, H=770, O=1001, r=5, dtype="f32", runs=90, p=0.1),
        # a block's residual at 128 x 1024 tokens
        dict(name="dropout_step", op="dropout_step", N=131072, H=1024, dtype="bf16", p=0.1, residual=True),
        # odd float32 rows
        dict(name="dropout_step_odd", op="dropout_step", N=4097, H=770, dtype="f32", p=0.25, residual=False),
        # a short step's input rows
        dict(name="dropout_short", op="dropout", N=320, H=1024, dtype="f16", p=0.1, residual=True),
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, even over its logarithm."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["sample", "sample", "adapters", "adapters", "adapters_step", "dropout", "dropout_step"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op == "sample":
        V = rng.choice([_log(rng, 1000, 160000), 8 * _log(rng, 125, 20000)])
        B = _log(rng, 1, max(1, min(256, 256 * 151936 // V)))
        return dict(op=op, B=B, V=V, dtype=dtype, settings=rng.choice(["none", "nucleus", "top_k", "mixed"]))
    H = rng.choice([_log(rng, 64, 4096), 64 * _log(rng, 1, 64)])
    if op in ("dropout", "dropout_step"):
        N = _log(rng, 1, max(1, min(131072, (1 << 27) // H)))
        return dict(op=op, N=N, H=H, dtype=dtype, p=rng.choice([0.05, 0.1, 0.5]), residual=rng.random() < 0.5)
    O = rng.choice([_log(rng, 64, 4096), 64 * _log(rng, 1, 64)])
    r = rng.choice([4, 8, 16, 16, 32, 64, rng.randint(1, 64)])
    A = _log(rng, 1, 16)
    N = _log(rng, 1, max(1, min(131072, (1 << 29) // ((H + O) * max(A, 4)))))
    case = dict(op=op, N=N, A=A, H=H, O=O, r=r, dtype=dtype, runs=rng.choice([1, 100, 1000]))
    return case if op == "adapters" else dict(case, p=rng.choice([0.0, 0.05]))


def _settings(kind, B, g):
    """Temperature, top_k, top_p, min_p: one number, or one a row."""
    if kind == "none":
        return dict(temperature=1.0, top_k=0, top_p=1.0, min_p=0.0)
    if kind == "nucleus":
        return dict(temperature=0.8, top_k=0, top_p=0.95, min_p=0.0)
    if kind == "top_k":
        return dict(temperature=0.7, top_k=50, top_p=0.9, min_p=0.0)

    def pick(values, dtype):
        at = torch.randint(0, len(values), (B,), generator=g, device="cuda")
        return torch.tensor(values, dtype=dtype, device="cuda")[at]

    return dict(temperature=pick([0.0, 0.6, 0.8, 1.0, 1.0, 1.3], torch.float32),
                top_k=pick([0, 0, 0, 20, 50, 1000], torch.int32),
                top_p=pick([1.0, 1.0, 0.9, 0.95, 0.99], torch.float32),
                min_p=pick([0.0, 0.0, 0.02, 0.1], torch.float32))


def _logits(shape, g):
    """Rows as a language model leaves them: a wide body, and a few tokens that hold most of the mass."""
    x = torch.randn(shape, generator=g, device="cuda") * 2.5
    top = torch.randint(0, shape[-1], (*shape[:-1], 12), generator=g, device="cuda")
    lift = 6.0 + 6.0 * torch.rand(top.shape, generator=g, device="cuda")
    return x.scatter_add_(-1, top, lift)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op, dt = case["op"], _DTYPES[case["dtype"]]

    def normal(*shape, size=1.0):
        return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).mul_(size).to(dt)

    if op == "sample":
        B, V = case["B"], case["V"]
        x = _logits((B, V), g).to(dt)
        return dict(case, x=x, u=torch.rand(B, generator=g, device="cuda"), args=_settings(case["settings"], B, g))
    N, H = case["N"], case["H"]
    state = dict(case, seed=seed * 7919 + 17, offset=seed % 1000)
    if op in ("dropout", "dropout_step"):
        state["x"] = normal(N, H)
        state["res"] = normal(N, H) if case["residual"] else None
        if op == "dropout_step":
            state["x"].requires_grad_()
            state["grad"] = normal(N, H, size=1e-3)
        return state
    A, O, r = case["A"], case["O"], case["r"]
    # tokens of a request stand together; one request in eight has no adapter (in training all have one)
    requests = -(-N // case["runs"])
    ids = torch.randint(0, A, (requests,), generator=g, device="cuda")
    if op == "adapters":
        ids = ids.masked_fill(torch.rand(requests, generator=g, device="cuda") < 0.125, -1)
    state["ids"] = ids.repeat_interleave(case["runs"])[:N].contiguous()
    state["x"] = normal(N, H)
    state["base"] = normal(N, O)
    state["down"] = normal(A, r, H, size=H ** -0.5)
    state["up"] = normal(A, O, r, size=0.1)
    state["scales"] = torch.full((A,), 32.0 / r, device="cuda")
    if op == "adapters_step":
        for k in ("x", "down", "up"):
            state[k].requires_grad_()
        state["grad"] = normal(N, O, size=1e-3)
    return state


def run(state):
    return _kernels(state) if own else _plain(state)


def _kernels(s):
    op = s["op"]
    if op == "sample":
        from rosellm_amd.roseinfer import sample_tokens

        out = sample_tokens(s["x"], s["u"], **s["args"])
        return dict(token_ids=out.token_ids, logprobs=out.logprobs, sampling_logprobs=out.sampling_logprobs)
    if op in ("dropout", "dropout_step"):
        from rosellm_amd.rosetrainer import dropout

        y = dropout(s["x"], s["p"], seed=s["seed"], offset=s["offset"], residual=s["res"])
        if op == "dropout":
            return y
        (dx,) = torch.autograd.grad(y, s["x"], s["grad"])
        return dict(out=y.detach(), dx=dx)
    from rosellm_amd.rosetrainer import adapter_linear

    if op == "adapters":
        return adapter_linear(s["x"], s["down"], s["up"], s["ids"], base=s["base"], scales=s["scales"])
    y = adapter_linear(s["x"], s["down"], s["up"], s["ids"], base=s["base"], scales=s["scales"],
                       dropout_p=s["p"], seed=s["seed"], offset=s["offset"])
    dx, ddown, dup = torch.autograd.grad(y, (s["x"], s["down"], s["up"]), s["grad"])
    return dict(out=y.detach(), dx=dx, ddown=ddown, dup=dup)


# ---- plain forms -------------------------------------------------------------


def _plain(s):
    op = s["op"]
    if op == "sample":
        return _sample(s["x"], s["u"], **s["args"])
    if op in ("dropout", "dropout_step"):
        x = s["x"].detach()
        keep = _keep(s, x.shape[0], x.shape[1], x.device)
        y = x.float() * keep
        if s["res"] is not None:
            y = y + s["res"].float()
        y = y.to(x.dtype)
        if op == "dropout":
            return y
        return dict(out=y, dx=(s["grad"].float() * keep).to(x.dtype))
    # the adapters side by side: every row's products with all of them, and zeros for all but its own
    x, down, up = s["x"].detach().float(), s["down"].detach().float(), s["up"].detach().float()
    A, r, H = down.shape
    dt = s["x"].dtype
    keep = None if op == "adapters" or s["p"] == 0.0 else _keep(s, x.shape[0], H, x.device)
    if keep is not None:
        x = x * keep
    mine = (s["ids"].unsqueeze(-1) == torch.arange(A, device=x.device)).float() * s["scales"]
    mine = mine.unsqueeze(-1).expand(-1, -1, r).reshape(-1, A * r)
    down, up = down.reshape(A * r, H), up.permute(0, 2, 1).reshape(A * r, -1)
    t = torch.mm(x, down.t()) * mine
    y = (s["base"].float() + torch.mm(t, up)).to(dt)
    if op == "adapters":
        return y
    g = s["grad"].float()
    t2 = torch.mm(g, up.t()) * mine
    dx = torch.mm(t2, down)
    if keep is not None:
        dx = dx * keep
    ddown = torch.mm(t2.t(), x).view(A, r, H)
    dup = torch.mm(t.t(), g).view(A, r, -1).permute(0, 2, 1).contiguous()
    return dict(out=y, dx=dx.to(dt), ddown=ddown.to(dt), dup=dup.to(dt))


def _sample(x, u, temperature, top_k, top_p, min_p):
    """In 64 bits: a token is taken, and an entry kept, where a running sum passes a border."""
    B, V = x.shape

    def column(v):
        return torch.as_tensor(v, dtype=torch.float64, device=x.device).expand(B).unsqueeze(-1)

    T, k, tp, mp = column(temperature), column(top_k), column(top_p), column(min_p)
    greedy = T <= 0
    T = torch.where(greedy, 1.0, T)
    xd = x.double()
    m = xd.amax(-1, keepdim=True)
    w = torch.exp((xd - m) / T)
    lse = w.sum(-1, keepdim=True).log()
    order = torch.sort(xd, dim=-1, descending=True, stable=True).indices
    rank = torch.arange(V, device=x.device)
    ws = w.gather(-1, order)
    ws = torch.where((k <= 0) | (rank < k), ws, 0.0)
    share = ws.cumsum(-1) / ws.sum(-1, keepdim=True)
    ws = torch.where((tp <= 0) | (tp >= 1) | (share <= tp) | (rank == 0), ws, 0.0)
    kept = torch.zeros_like(w).scatter_(-1, order, ws)
    kept = torch.where(xd - m >= T * mp.clamp(0.0, 1.0).log(), kept, 0.0)
    first = torch.where(rank == order[:, :1], 1.0, 0.0)
    kept = torch.where(greedy, first, kept)
    total = kept.cumsum(-1)
    token = (total > u.double().unsqueeze(-1) * total[:, -1:]).long().argmax(-1, keepdim=True)
    lp = (xd - m).gather(-1, token) / T - lse
    lq = torch.where(greedy, 0.0, kept.gather(-1, token).log() - total[:, -1:].log())
    return dict(token_ids=token.squeeze(-1), logprobs=lp.squeeze(-1).float(), sampling_logprobs=lq.squeeze(-1).float())


def _keep(s, N, H, device):
    """What each entry is multiplied by: 0 or 1 / (1 - p), p in steps of 2^-16. The counter is the group's index and
    the offset; half a word an entry, the low half first."""
    M = 0xFFFFFFFF
    groups = -(-H // _GROUP)
    i = torch.arange(N * groups, device=device)
    c0, c1 = i & M, i >> 32
    c2 = torch.full_like(i, s["offset"] & M)
    c3 = torch.full_like(i, s["offset"] >> 32)
    k0, k1 = s["seed"] & M, s["seed"] >> 32
    for _ in range(10):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = ((b >> 32) & M) ^ c1 ^ k0, b & M, ((a >> 32) & M) ^ c3 ^ k1, a & M
        k0, k1 = (k0 + 0x9E3779B9) & M, (k1 + 0xBB67AE85) & M
    half = torch.stack([c0 & 0xFFFF, c0 >> 16, c1 & 0xFFFF, c1 >> 16, c2 & 0xFFFF, c2 >> 16, c3 & 0xFFFF, c3 >> 16], -1)
    cut = round(s["p"] * 65536)
    return torch.where(half >= cut, 65536.0 / (65536 - cut), 0.0).view(N, groups * _GROUP)[:, :H]


# ---- what each cannot do without, and its 64-bit results ------------------------


def work(case):
    op, size = case["op"], _SIZES[case["dtype"]]
    if op == "sample":
        n = case["B"] * case["V"]
        # an exponential and a sum an entry
        return {"bytes": n * size + case["B"] * 36, "flops": 2 * n}
    N, H = case["N"], case["H"]
    if op in ("dropout", "dropout_step"):
        n = N * H * (3 if case["residual"] else 2) + (2 * N * H if op == "dropout_step" else 0)
        return {"bytes": n * size, "flops": n}
    A, O, r = case["A"], case["O"], case["r"]
    # adapters of requests that are in the batch
    used = A * (1.0 - (1.0 - 1.0 / A) ** -(-N // case["runs"])) if A > 1 else 1
    weights = round(used * r * (H + O))
    fwd = (N * (H + 2 * O) + weights) * size + 8 * N
    if op == "adapters":
        return {"bytes": fwd, "flops": 2 * N * r * (H + O)}
    return {"bytes": fwd + (N * (O + H) + A * r * (H + O)) * size, "flops": 6 * N * r * (H + O)}


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "sample":
        return _exact_sample(s)
    if op in ("dropout", "dropout_step"):
        keep = _exact_keep(s, case["N"], case["H"])
        y = torch.zeros(keep.shape, dtype=torch.float64, device="cuda") if s["res"] is None else s["res"].double()
        y = torch.addcmul(y, s["x"].detach().double(), keep)
        return y if op == "dropout" else dict(out=y, dx=s["grad"].double().mul_(keep))
    x, down, up = s["x"].detach(), s["down"].detach().double(), s["up"].detach().double()
    step = op == "adapters_step"
    keep = _exact_keep(s, case["N"], case["H"]) if step and s["p"] > 0 else None
    y = s["base"].double()
    dx = torch.zeros(x.shape, dtype=torch.float64, device="cuda") if step else None
    ddown, dup = torch.zeros_like(down), torch.zeros_like(up)
    for a in range(case["A"]):
        rows = torch.nonzero(s["ids"] == a).flatten()
        if rows.numel() == 0:
            continue
        scale = float(s["scales"][a])
        xa = x[rows].double()
        if keep is not None:
            xa *= keep[rows]
        t = xa @ down[a].T.contiguous()
        y[rows] += scale * (t @ up[a].T.contiguous())
        if step:
            g = s["grad"][rows].double()
            back = scale * (g @ up[a])
            ddown[a] = back.T.contiguous() @ xa
            dup[a] = scale * (g.T.contiguous() @ t)
            back = back @ down[a]
            dx[rows] = back if keep is None else back * keep[rows]
    return dict(out=y, dx=dx, ddown=ddown, dup=dup) if step else y


def _exact_sample(s):
    """Row by row, over the entries in descending order."""
    B, V = s["x"].shape
    ids = torch.zeros(B, dtype=torch.int64, device="cuda")
    lps = torch.zeros(B, dtype=torch.float64, device="cuda")
    lqs = torch.zeros(B, dtype=torch.float64, device="cuda")
    args = {n: torch.as_tensor(v, dtype=torch.float64).expand(B).tolist() if not torch.is_tensor(v) else v.double().tolist()
            for n, v in s["args"].items()}
    for b in range(B):
        T, k, tp, mp = (args[n][b] for n in ("temperature", "top_k", "top_p", "min_p"))
        x = s["x"][b].to(torch.float64)
        if T <= 0:
            z = x - torch.logsumexp(x, 0)
            ids[b] = torch.nonzero(x == x.max())[0, 0]
            lps[b] = z[ids[b]]
            continue
        z = x / T
        z = z - torch.logsumexp(z, 0)
        value, at = torch.sort(z, descending=True, stable=True)
        n = int(k) if 0 < k < V else V
        if 0.0 < tp < 1.0:
            mass = value[:n].exp()
            mass = mass.cumsum(0).div(mass.sum())
            n = max(1, int((mass <= tp).sum()))
        if mp > 0.0:
            n = min(n, int((x[at] - x.max() >= T * math.log(min(mp, 1.0))).sum()))
        chosen = torch.sort(at[:n]).values
        mass = torch.cumsum(z[chosen].exp(), 0)
        i = int(torch.searchsorted(mass, s["u"][b].double() * mass[-1], right=True))
        ids[b] = chosen[i]
        lps[b] = z[chosen[i]]
        lqs[b] = z[chosen[i]] - mass[-1].log()
    return dict(token_ids=ids, logprobs=lps, sampling_logprobs=lqs)


def _exact_keep(s, N, H):
    """The generator by its definition on four words, with products from 16-bit halves."""
    word = 2 ** 32

    def product(a, m):
        """High and low words of a * m."""
        low = (a % 65536) * m
        high = (a // 65536) * m + low // 65536
        return high // 65536, (high % 65536) * 65536 + low % 65536

    groups = (H + _GROUP - 1) // _GROUP
    n = torch.arange(N * groups, dtype=torch.int64, device="cuda")
    c = [n % word, n // word, torch.full_like(n, s["offset"] % word), torch.full_like(n, s["offset"] // word)]
    key = [s["seed"] % word, s["seed"] // word]
    for _ in range(10):
        h0, l0 = product(c[0], 0xD2511F53)
        h1, l1 = product(c[2], 0xCD9E8D57)
        c = [h1 ^ c[1] ^ key[0], l1, h0 ^ c[3] ^ key[1], l0]
        key = [(key[0] + 0x9E3779B9) % word, (key[1] + 0xBB67AE85) % word]
    cut = round(s["p"] * 65536)
    keep = torch.empty((N, groups, _GROUP), dtype=torch.float64, device="cuda")
    for j in range(_GROUP):
        bits = c[j // 2] // (65536 if j % 2 else 1) % 65536
        keep[:, :, j] = (bits.view(N, groups) >= cut).double() * (65536.0 / (65536 - cut))
    return keep.view(N, groups * _GROUP)[:, :H]
