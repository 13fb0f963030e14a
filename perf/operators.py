"""Operators of a speculative rollout step, and of the training step that its
tokens feed, as they are measured: the calls of a user's program, their
inputs, their plain form in elementary torch operations, what each cannot do
without, and their 64-bit results.

* ``verify``: drafted tokens against the target's distribution, from given
  uniforms (``rosellm_amd.roseinfer.verify_draft_tokens``).
* ``quantize``: a matrix into microscaled 4-bit floating point and back
  (``quantize_mxfp4``, ``dequantize_mxfp4``).
* ``head``: a draft model's logits from a head held in 4 bits
  (``mxfp4_linear``).
* ``embed`` / ``embed_step``: the scaled embedding lookup, and with its
  gradient (``rosellm_amd.rosetrainer.embedding``).
"""

import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_SIZES = {"bf16": 2, "f16": 2, "f32": 4}

# The entries of one microscaled block, and what a row of blocks is padded to.
_BLOCK, _DEPTH = 32, 128


def listed():
    return [
        # one sequence of a low-latency rollout, four drafted tokens
        dict(name="verify_one", op="verify", B=1, K=4, V=151936, dtype="bf16", T=1.0, ragged=False, q=True),
        # a rollout batch, sampled a little below temperature 1
        dict(name="verify_batch", op="verify", B=64, K=5, V=151936, dtype="bf16", T=0.8, ragged=False, q=True),
        # float32 logits of an odd vocabulary, drafts of different lengths
        dict(name="verify_ragged_f32", op="verify", B=37, K=3, V=50257, dtype="f32", T=1.0, ragged=True, q=True),
        # drafts copied from the prompt (no draft model, so no draft logits)
        dict(name="verify_copied", op="verify", B=16, K=7, V=151936, dtype="bf16", T=1.0, ragged=True, q=False),
        # the draft head after a policy update
        dict(name="quantize_head", op="quantize", R=151936, H=1024, dtype="bf16"),
        # a small odd matrix whose rows end inside a block
        dict(name="quantize_odd", op="quantize", R=777, H=1000, dtype="f32"),
        # one decode step of a few sequences' draft model
        dict(name="head_decode", op="head", M=8, V=151936, H=1024, dtype="bf16"),
        # a full decode batch on a wide, odd head
        dict(name="head_batch_odd", op="head", M=130, V=50257, H=2080, dtype="bf16"),
        # draft logits of whole prompts
        dict(name="head_prompt", op="head", M=2048, V=151936, H=1024, dtype="bf16"),
        # the input rows of the verified tokens of one decode step, rejected places padded
        dict(name="embed_decode", op="embed", N=320, V=151936, H=1024, dtype="bf16", scale=32.0, pad=0.4),
        # the policy's training step at 256 x 1024 tokens
        dict(name="embed_step", op="embed_step", N=262144, V=151936, H=1024, dtype="bf16", scale=1.0, pad=0.1),
        # a short float32 step of odd sizes
        dict(name="embed_step_odd", op="embed_step", N=4097, V=50257, H=770, dtype="f32", scale=27.75, pad=0.0),
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, even over its logarithm."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["verify", "verify", "quantize", "head", "head", "embed", "embed_step"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    V = rng.choice([_log(rng, 1000, 160000), 8 * _log(rng, 125, 20000)])
    H = rng.choice([_log(rng, 64, 4096), 64 * _log(rng, 1, 64)])
    if op == "verify":
        K = rng.randint(1, 8)
        B = _log(rng, 1, max(1, min(96, 64 * 11 * 151936 // ((2 * K + 1) * V))))
        return dict(op=op, B=B, K=K, V=V, dtype=dtype, T=rng.choice([1.0, 1.0, 0.6, 1.3]),
                    ragged=rng.random() < 0.5, q=rng.random() < 0.75)
    if op == "quantize":
        return dict(op=op, R=_log(rng, 1, max(1, min(160000, (1 << 28) // H))), H=H, dtype=dtype)
    if op == "head":
        return dict(op=op, M=_log(rng, 1, max(1, min(2048, (1 << 31) // (V * max(H // 512, 1))))), V=V, H=H,
                    dtype=dtype)
    N = _log(rng, 1, max(1, min(262144, (1 << 28) // H)))
    return dict(op=op, N=N, V=V, H=H, dtype=dtype, scale=rng.choice([1.0, math.sqrt(H)]),
                pad=rng.choice([0.0, 0.3]))


def _logits(shape, g):
    """Rows as a language model leaves them: a wide body, and a few tokens that hold most of the mass."""
    x = torch.randn(shape, generator=g, device="cuda") * 2.5
    top = torch.randint(0, shape[-1], (*shape[:-1], 12), generator=g, device="cuda")
    lift = 6.0 + 6.0 * torch.rand(top.shape, generator=g, device="cuda")
    return x.scatter_add_(-1, top, lift)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op, dt = case["op"], _DTYPES[case["dtype"]]
    if op == "verify":
        B, K, V, T = case["B"], case["K"], case["V"], case["T"]
        x = _logits((B, K + 1, V), g)
        y = x[:, :K] + 0.7 * torch.randn((B, K, V), generator=g, device="cuda")
        y = y.to(dt)
        # drafts are sampled from the draft's distribution
        noise = torch.rand((B, K, V), generator=g, device="cuda").clamp_min_(1e-30).log_().neg_().log_().neg_()
        tokens = noise.add_(y, alpha=1.0 / T).argmax(-1)
        if case["ragged"]:
            n = torch.randint(0, K + 1, (B, 1), generator=g, device="cuda")
            tokens = tokens.masked_fill(torch.arange(K, device="cuda") >= n, -1)
        return dict(case, target=x.to(dt), draft=y if case["q"] else None, tokens=tokens,
                    uniforms=torch.rand((B, K + 1), generator=g, device="cuda"))
    if op == "quantize":
        x = torch.randn((case["R"], case["H"]), generator=g, device="cuda")
        x *= 0.02 * torch.exp(0.5 * torch.randn((1, case["H"]), generator=g, device="cuda"))
        return dict(case, x=x.to(dt))
    if op == "head":
        # normalised hidden states with a few large channels; the head is kept in 4 bits
        M, V, H = case["M"], case["V"], case["H"]
        x = torch.randn((M, H), generator=g, device="cuda")
        x *= torch.exp(0.7 * torch.randn((1, H), generator=g, device="cuda"))
        codes, scales = _quantize(0.05 * torch.randn((V, H), generator=g, device="cuda"))
        return dict(case, x=x.to(dt), codes=codes, scales=scales)
    N, V, H = case["N"], case["V"], case["H"]
    # token frequencies fall off as one over the rank, at ids in no order
    rank = torch.exp(torch.rand(N, generator=g, device="cuda") * math.log(V)).long().clamp_(1, V) - 1
    ids = torch.randperm(V, generator=g, device="cuda")[rank]
    ids = ids.masked_fill(torch.rand(N, generator=g, device="cuda") < case["pad"], -1)
    weight = (0.02 * torch.randn((V, H), generator=g, device="cuda")).to(dt)
    state = dict(case, ids=ids, weight=weight)
    if op == "embed_step":
        weight.requires_grad_()
        state["grad"] = (1e-3 * torch.randn((N, H), generator=g, device="cuda")).to(dt)
    return state


def run(state):
    return _kernels(state) if own else _plain(state)


def _kernels(s):
    op = s["op"]
    if op == "verify":
        from rosellm_amd.roseinfer import verify_draft_tokens

        out = verify_draft_tokens(s["target"], s["tokens"], s["draft"], s["uniforms"], s["T"])
        return dict(token_ids=out.token_ids, num_accepted=out.num_accepted, logprobs=out.logprobs)
    if op == "quantize":
        from rosellm_amd.roseinfer import dequantize_mxfp4, quantize_mxfp4

        return dequantize_mxfp4(quantize_mxfp4(s["x"]), torch.bfloat16)
    if op == "head":
        from rosellm_amd.roseinfer import MxFp4, mxfp4_linear

        return mxfp4_linear(s["x"], MxFp4(s["codes"], s["scales"], s["H"]))
    from rosellm_amd.rosetrainer import embedding

    if op == "embed":
        return embedding(s["ids"], s["weight"], scale=s["scale"], padding_idx=-1)
    out = embedding(s["ids"], s["weight"], scale=s["scale"], padding_idx=-1)
    (dw,) = torch.autograd.grad(out, s["weight"], s["grad"])
    return dict(out=out.detach(), dweight=dw)


# ---- plain forms -------------------------------------------------------------


def _quantize(x):
    """Microscaled 4-bit blocks of the rows of x [R, H]: codes [R, P / 2] (two entries a byte, the first in the low
    half) and scales [R, P / 32], P = H rounded up to a multiple of 128 with blocks of zeros."""
    R, H = x.shape
    P = -(-H // _DEPTH) * _DEPTH
    v = torch.nn.functional.pad(x.float(), (0, P - H)).view(R, P // _BLOCK, _BLOCK)
    amax = v.abs().amax(-1, keepdim=True)
    # amax = m 2^e with m in [1/2, 1), so that the largest power of two in it is 2^(e - 1); 4 is that of the format
    e = torch.where(amax > 0, torch.frexp(amax).exponent - 3, -127).clamp(-127, 127)
    a = v * ((127 - e).clamp(1, 254) << 23).to(torch.int32).view(torch.float32)
    b = a.abs()
    # round to nearest, ties to the even code, of 0, 0.5, 1, 1.5, 2, 3, 4, 6
    code = ((b > 0.25).to(torch.uint8) + (b >= 0.75) + (b > 1.25) + (b >= 1.75) + (b > 2.5) + (b >= 3.5) + (b > 5.0))
    code = (code + 8 * torch.signbit(a).to(torch.uint8)).view(R, P // 2, 2)
    return code[..., 0] + 16 * code[..., 1], (e.squeeze(-1) + 127).to(torch.uint8)


def _values(codes, scales, H, dtype):
    """The numbers that the blocks stand for, [R, H]."""
    R = codes.shape[0]
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=codes.device, dtype=dtype)
    grid = torch.cat([grid, -grid])
    v = grid[torch.stack([codes & 15, codes >> 4], -1).long()].view(R, -1, _BLOCK)
    unit = torch.exp2(scales.to(dtype).unsqueeze(-1) - 127.0)
    return (v * unit).view(R, -1)[:, :H]


def _plain(s):
    op = s["op"]
    if op == "verify":
        return _verify(s["target"], s["tokens"], s["draft"], s["uniforms"], s["T"])
    if op == "quantize":
        codes, scales = _quantize(s["x"])
        return _values(codes, scales, s["H"], torch.float32).to(torch.bfloat16)
    if op == "head":
        x = _values(*_quantize(s["x"]), s["H"], torch.float32)
        w = _values(s["codes"], s["scales"], s["H"], torch.float32)
        return torch.mm(x, w.t()).to(s["x"].dtype)
    ids, weight = s["ids"], s["weight"].detach()
    here = (ids >= 0).unsqueeze(-1)
    out = torch.where(here, weight[ids.clamp_min(0)].float() * s["scale"], 0.0).to(weight.dtype)
    if op == "embed":
        return out
    # sums of up to some ten thousand gradients of one token: held in 64 bits
    order = torch.sort(ids, stable=True).indices
    part = torch.where(here[order], s["grad"][order].double(), 0.0)
    dw = torch.zeros(weight.shape, dtype=torch.float64, device=weight.device)
    dw.index_add_(0, ids[order].clamp_min(0), part)
    return dict(out=out, dweight=(dw * s["scale"]).to(weight.dtype))


def _softmax(x, T):
    z = x.double() / T
    z = torch.exp(z - z.amax(-1, keepdim=True))
    return z / z.sum(-1, keepdim=True)


def _verify(target, tokens, draft, uniforms, T):
    """In 64 bits: a token is taken where a running sum passes a border."""
    B, K = tokens.shape
    u = uniforms.double()
    p = _softmax(target, T)
    at = tokens.clamp_min(0).unsqueeze(-1)
    px = p[:, :K].gather(-1, at).squeeze(-1)
    if draft is None:
        q = torch.zeros_like(p[:, :K]).scatter_(-1, at, 1.0)
    else:
        q = _softmax(draft, T)
    qx = q.gather(-1, at).squeeze(-1)
    drafted = (tokens >= 0).long().cumprod(-1)
    n = ((u[:, :K] * qx < px).long() * drafted).cumprod(-1).sum(-1)
    rejected = n < drafted.sum(-1)
    row = torch.arange(B, device=p.device)
    pn = p[row, n]
    rest = (pn - q[row, n.clamp_max(K - 1)]).clamp_min(0.0)
    rest = torch.where((rejected & (rest.sum(-1) > 0)).unsqueeze(-1), rest, pn)
    run_ = rest.cumsum(-1)
    last = (run_ > u[:, K:] * run_[:, -1:]).long().argmax(-1)
    j = torch.arange(K + 1, device=p.device)
    ids = torch.cat([tokens, tokens.new_full((B, 1), -1)], 1).masked_fill(j > n.unsqueeze(-1), -1)
    ids[row, n] = last
    lp = p.gather(-1, ids.clamp_min(0).unsqueeze(-1)).squeeze(-1).log().masked_fill(ids < 0, 0.0)
    return dict(token_ids=ids, num_accepted=n, logprobs=lp.float())


# ---- what each cannot do without, and its 64-bit results ------------------------


def work(case):
    op, size = case["op"], _SIZES[case["dtype"]]
    if op == "verify":
        rows = case["B"] * (case["K"] + 1 + (case["K"] if case["q"] else 0))
        # an exponential and a sum an entry
        return {"bytes": rows * case["V"] * size + case["B"] * (case["K"] + 1) * 24, "flops": 2 * rows * case["V"]}
    if op == "quantize":
        n = case["R"] * case["H"]
        return {"bytes": n * (size + 2) + n * 17 // 32, "flops": 3 * n}
    if op == "head":
        M, V, H = case["M"], case["V"], case["H"]
        return {"bytes": M * H * size + V * H * 17 // 32 + M * V * size, "flops": 2 * M * V * H}
    N, V, H = case["N"], case["V"], case["H"]
    kept = round(N * (1.0 - case["pad"]))
    # the ids' distinct rows are read once; a rank's frequency is 1 / (rank log V)
    seen = min(kept, V)
    fwd = seen * H * size + N * H * size + 8 * N
    if op == "embed":
        return {"bytes": fwd, "flops": N * H}
    return {"bytes": fwd + kept * H * size + V * H * size, "flops": 2 * N * H}


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "verify":
        # row by row: log-probabilities by log-sum-exp, the draw by a search in the running sum
        T, K = case["T"], case["K"]
        ids = torch.full((case["B"], K + 1), -1, device="cuda")
        lps = torch.zeros((case["B"], K + 1), dtype=torch.float64, device="cuda")
        count = torch.zeros(case["B"], dtype=torch.int64, device="cuda")
        for b in range(case["B"]):
            j, rest = 0, None
            while True:
                z = s["target"][b, j].to(torch.float64).div(T)
                lp = z - torch.logsumexp(z, 0)
                d = int(s["tokens"][b, j]) if j < K else -1
                if d < 0:
                    rest = lp.exp()
                    break
                if case["q"]:
                    z = s["draft"][b, j].to(torch.float64).div(T)
                    lq = z - torch.logsumexp(z, 0)
                else:
                    lq = torch.full_like(lp, -math.inf)
                    lq[d] = 0.0
                if float(s["uniforms"][b, j]) < math.exp(float(lp[d] - lq[d])):
                    ids[b, j], lps[b, j], j = d, lp[d], j + 1
                    continue
                rest = torch.relu(lp.exp() - lq.exp())
                break
            total = torch.cumsum(rest, 0)
            t = int(torch.searchsorted(total, s["uniforms"][b, K].double() * total[-1], right=True))
            ids[b, j], lps[b, j], count[b] = t, lp[t], j
        return dict(token_ids=ids, num_accepted=count, logprobs=lps)
    if op == "quantize":
        return _near(s["x"])[:, : case["H"]]
    if op == "head":
        x = _near(s["x"])[:, : case["H"]]
        low, high = s["codes"] % 16, s["codes"] // 16
        code = torch.empty((case["V"], 2 * low.shape[1]), dtype=torch.int64, device="cuda")
        code[:, 0::2], code[:, 1::2] = low.long(), high.long()
        # sign, exponent (2 bits, bias 1), mantissa (1 bit)
        sign, e, m = 1.0 - 2.0 * (code // 8), (code // 2) % 4, (code % 2).double()
        size = torch.where(e > 0, torch.pow(2.0, (e - 1).double()) * (1.0 + m / 2), m / 2)
        unit = torch.pow(2.0, s["scales"].double() - 127.0).repeat_interleave(_BLOCK, 1)
        return torch.matmul(x, (sign * size * unit)[:, : case["H"]].T)
    scale, ids = case["scale"], s["ids"]
    w = s["weight"].detach()
    out = torch.zeros((case["N"], case["H"]), dtype=torch.float64, device="cuda")
    some = torch.nonzero(ids >= 0).flatten()
    out[some] = w[ids[some]].double() * scale
    if op == "embed":
        return out
    # the sums as differences of running sums of the sorted rows
    key, order = torch.sort(ids[some])
    total = torch.zeros((some.numel() + 1, case["H"]), dtype=torch.float64, device="cuda")
    torch.cumsum(s["grad"][some[order]].double(), 0, out=total[1:])
    v = torch.arange(case["V"], device="cuda")
    lo, hi = torch.searchsorted(key, v), torch.searchsorted(key, v, right=True)
    return dict(out=out, dweight=(total[hi] - total[lo]) * scale)


def _near(x):
    """Each entry's nearest number of its block's grid, by distances, ties to the even code."""
    R, H = x.shape
    v = torch.nn.functional.pad(x.double(), (0, -H % _BLOCK)).view(R, -1, _BLOCK)
    amax = v.abs().amax(-1, keepdim=True)
    top = amax.clamp_min(2.0 ** -125)
    unit = top / torch.frexp(top).mantissa / 8.0  # a quarter of the largest power of two in it
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64, device=x.device)
    a = v.abs() / unit
    # between two neighbours the nearer one; halfway the one of even index
    above = torch.searchsorted(grid, a.contiguous()).clamp_max(7)
    below = (above - 1).clamp_min(0)
    up, down = grid[above] - a, a - grid[below]
    pick = torch.where((up < down) | ((up == down) & (above % 2 == 0)), above, below)
    return (grid[pick] * torch.sign(v) * unit).view(R, -1)
