"""Workloads of the token operators (layer norm, attention over packed clouds, attention of single
tokens over a cache): their inputs, their plain form in elementary torch operations, the calls that a
user makes of this package, the work that a pass cannot do without, and the results in 64 bits.

`own` chooses what run() does: False, the plain form in 32 bits; True, this package's operators.
Lengths of clouds come from the case (`lengths` seeds them), values from prepare()'s seed.
"""
import math
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
DEVICE = "cuda"


def listed():
    return [
        # the tokens of one small cloud between two layers: latency counts
        {"name": "norm_tokens_small", "op": "norm", "train": False, "dtype": "f32", "rows": 96, "width": 384},
        # a serving batch's activations, streamed once
        {"name": "norm_wide_bf16", "op": "norm", "train": False, "dtype": "bf16", "rows": 32768, "width": 1024},
        # per-point features of a batch of 8 clouds of 8192 points, one training step
        {"name": "norm_train_points", "op": "norm", "train": True, "dtype": "f32", "rows": 65536, "width": 512},
        # odd width and row count: no alignment to lean on
        {"name": "norm_train_odd_f16", "op": "norm", "train": True, "dtype": "f16", "rows": 10007, "width": 771},
        # a few new tokens of four small clouds against their own and earlier ones
        {"name": "packed_small_f32", "op": "packed", "train": False, "dtype": "f32", "clouds": 4, "shortest": 1,
         "longest": 64, "prefix": 40, "heads": 6, "kv_heads": 6, "width": 64, "causal": True, "lengths": 1},
        # whole prompts, grouped heads
        {"name": "packed_prompt_bf16", "op": "packed", "train": False, "dtype": "bf16", "clouds": 3, "shortest": 4096,
         "longest": 8192, "prefix": 0, "heads": 16, "kv_heads": 4, "width": 128, "causal": True, "lengths": 2},
        # training on many clouds of very different sizes in one packed batch
        {"name": "packed_train_ragged", "op": "packed", "train": True, "dtype": "bf16", "clouds": 16, "shortest": 50,
         "longest": 2048, "prefix": 0, "heads": 12, "kv_heads": 12, "width": 64, "causal": True, "lengths": 3},
        # training on two large clouds, every token sees every token
        {"name": "packed_train_large", "op": "packed", "train": True, "dtype": "f16", "clouds": 2, "shortest": 4096,
         "longest": 8192, "prefix": 0, "heads": 16, "kv_heads": 8, "width": 128, "causal": False, "lengths": 4},
        # training in 32 bits, the default type of a point cloud
        {"name": "packed_train_f32", "op": "packed", "train": True, "dtype": "f32", "clouds": 8, "shortest": 100,
         "longest": 1024, "prefix": 0, "heads": 6, "kv_heads": 6, "width": 64, "causal": False, "lengths": 5},
        # one token of one short generation: latency counts
        {"name": "cached_one_f16", "op": "cached", "dtype": "f16", "clouds": 1, "shortest": 700, "longest": 1024,
         "heads": 8, "kv_heads": 8, "width": 64, "lengths": 6},
        # one token each for a serving batch of ragged caches, grouped heads
        {"name": "cached_batch_bf16", "op": "cached", "dtype": "bf16", "clouds": 64, "shortest": 1, "longest": 8192,
         "heads": 32, "kv_heads": 8, "width": 128, "lengths": 7},
        # one token over one very long cache: the long axis has to be split
        {"name": "cached_long_f16", "op": "cached", "dtype": "f16", "clouds": 1, "shortest": 131072, "longest": 131072,
         "heads": 16, "kv_heads": 4, "width": 128, "lengths": 8},
    ]


def _between(rng, low, high):
    """A whole number of [low, high], spread over its logarithm."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def _size(n):
    return n + 1 if n == 3072 else n


def draw(rng):
    kind = rng.choice(("norm", "norm_train", "packed", "packed_train", "cached", "cached"))
    if kind.startswith("norm"):
        dtype = rng.choice(("f32", "f16", "bf16"))
        width = _size(_between(rng, 32, 8192))
        if rng.random() < 0.7:
            width = _size(-(-width // 8) * 8)
        rows = _size(_between(rng, 1, max(1, min(65536, 32 * 1024 * 1024 // width))))
        return {"op": "norm", "train": kind == "norm_train", "dtype": dtype, "rows": rows, "width": width}
    heads = rng.choice((4, 6, 8, 12, 16))
    kv_heads = heads // rng.choice([g for g in (1, 2, 4, 8) if heads % g == 0])
    width = rng.choice((32, 40, 64, 64, 80, 96, 128, 128))
    if kind.startswith("packed"):
        train = kind == "packed_train"
        dtype = rng.choice(("f32", "f16", "bf16", "bf16"))
        clouds = _between(rng, 1, 48)
        # the plain form holds (clouds, heads, longest, longest) scores in 32 bits
        most = int(math.sqrt((3e8 if dtype == "f32" else 1e9) / (clouds * heads)))
        longest = _size(_between(rng, 8, max(16, min(8192, most))))
        shortest = max(1, int(longest * rng.choice((0.02, 0.3, 0.9))))
        prefix = 0 if train or rng.random() < 0.6 else _size(_between(rng, 1, longest))
        return {"op": "packed", "train": train, "dtype": dtype, "clouds": clouds, "shortest": shortest,
                "longest": longest, "prefix": prefix, "heads": heads, "kv_heads": kv_heads, "width": width,
                "causal": rng.random() < 0.6, "lengths": rng.randrange(1 << 20)}
    dtype = rng.choice(("f32", "f16", "bf16", "bf16"))
    clouds = _between(rng, 1, 64)
    longest = _size(_between(rng, 16, min(131072, 64 * 4096 * 8 * 128 * 2 // (clouds * kv_heads * width * SIZE[dtype]))))
    shortest = max(1, int(longest * rng.choice((0.02, 0.5, 1.0))))
    return {"op": "cached", "dtype": dtype, "clouds": clouds, "shortest": shortest, "longest": longest,
            "heads": heads, "kv_heads": kv_heads, "width": width, "lengths": rng.randrange(1 << 20)}


def _lengths(case):
    """Tokens of each cloud, and keys of each cloud (its tokens and those before them)."""
    r = random.Random(case["lengths"])
    q = [r.randint(case["shortest"], case["longest"]) for _ in range(case["clouds"])]
    k = [n + (r.randint(0, case["prefix"]) if case.get("prefix") else 0) for n in q]
    return q, k


def _offsets(lengths):
    at = [0]
    for n in lengths:
        at.append(at[-1] + n)
    return torch.tensor(at, dtype=torch.int64).to(DEVICE)


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(int(seed))
    dtype = DTYPES[case["dtype"]]

    def rand(*shape):
        return torch.randn(*shape, generator=g, device=DEVICE, dtype=torch.float32).to(dtype)

    state = {"case": case, "train": bool(case.get("train"))}
    if case["op"] == "norm":
        rows, width = case["rows"], case["width"]
        # features with an offset and a spread of their own in each row
        x = torch.randn(rows, width, generator=g, device=DEVICE)
        x = x * (0.5 + torch.rand(rows, 1, generator=g, device=DEVICE)) + torch.randn(rows, 1, generator=g, device=DEVICE)
        state.update(x=x.to(dtype), weight=(1 + 0.1 * rand(width).float()).to(dtype), bias=0.1 * rand(width), eps=1e-5)
        if state["train"]:
            state["dy"] = rand(rows, width)
            for name in ("x", "weight", "bias"):
                state[name].requires_grad_()
        return state
    h, hk, d = case["heads"], case["kv_heads"], case["width"]
    lq, lk = _lengths(case)
    if case["op"] == "packed":
        state.update(q=rand(sum(lq), h, d), k=rand(sum(lk), hk, d), v=rand(sum(lk), hk, d), offsets=_offsets(lq),
                     offsets_k=_offsets(lk) if case["prefix"] else None, longest_q=max(lq), longest_k=max(lk))
        if state["train"]:
            state["do"] = rand(sum(lq), h, d)
            for name in ("q", "k", "v"):
                state[name].requires_grad_()
        return state
    n, p = case["clouds"], case["longest"]
    state.update(q=rand(n, h, d), k=rand(n, p, hk, d), v=rand(n, p, hk, d),
                 lengths=torch.tensor(lq, dtype=torch.int64).to(DEVICE))
    return state


def _norm_plain(s):
    with torch.no_grad():
        dtype = s["x"].dtype
        x, w, b = s["x"].float(), s["weight"].float(), s["bias"].float()
        centred = x - x.mean(1, keepdim=True)
        rstd = (centred.square().mean(1, keepdim=True) + s["eps"]).rsqrt()
        unit = centred * rstd
        y = (unit * w + b).to(dtype)
        if not s["train"]:
            return {"y": y}
        dy = s["dy"].float()
        du = dy * w
        dx = rstd * (du - du.mean(1, keepdim=True) - unit * (du * unit).mean(1, keepdim=True))
        return {"y": y, "dx": dx.to(dtype), "dweight": (dy * unit).sum(0).to(dtype), "dbias": dy.sum(0).to(dtype)}


def _to_clouds(x, offsets, longest):
    """(tokens, heads, width) packed -> (clouds, heads, longest, width) in 32 bits, zeros beyond each cloud's end."""
    at = torch.arange(longest, device=x.device)
    here = at[None, :] < (offsets[1:] - offsets[:-1])[:, None]
    index = (offsets[:-1, None] + at).clamp(max=x.shape[0] - 1)
    return (x[index].float() * here[:, :, None, None]).transpose(1, 2)


def _to_packed(x, offsets, tokens, dtype):
    """The reverse of _to_clouds, from (clouds, heads, longest, width)."""
    t = torch.arange(tokens, device=x.device)
    cloud = torch.searchsorted(offsets, t, right=True) - 1
    return x[cloud, :, t - offsets[cloud]].to(dtype)


def _packed_plain(s):
    with torch.no_grad():
        case, offsets = s["case"], s["offsets"]
        offsets_k = offsets if s["offsets_k"] is None else s["offsets_k"]
        dtype, (t, h, d), (tk, hk, _) = s["q"].dtype, s["q"].shape, s["k"].shape
        n, lq, lk = case["clouds"], s["longest_q"], s["longest_k"]
        scale = 1 / math.sqrt(d)
        q = _to_clouds(s["q"], offsets, lq).reshape(n, hk, h // hk * lq, d)
        k, v = _to_clouds(s["k"], offsets_k, lk), _to_clouds(s["v"], offsets_k, lk)
        len_q, len_k = offsets[1:] - offsets[:-1], offsets_k[1:] - offsets_k[:-1]
        i, j = torch.arange(lq, device=DEVICE)[None, :, None], torch.arange(lk, device=DEVICE)[None, None, :]
        seen = (i < len_q[:, None, None]) & (j < len_k[:, None, None])
        if case["causal"]:
            seen = seen & (j <= i + (len_k - len_q)[:, None, None])
        hidden = ~seen[:, None, None]
        p = (q @ k.transpose(2, 3)).reshape(n, hk, h // hk, lq, lk).mul_(scale).masked_fill_(hidden, -math.inf)
        top = p.amax(-1, keepdim=True)
        p = p.sub_(top.masked_fill(top == -math.inf, 0)).exp_()
        p = p.div_(p.sum(-1, keepdim=True).clamp_(min=1e-30)).reshape(n, hk, h // hk * lq, lk)
        o = p @ v
        out = {"o": _to_packed(o.reshape(n, h, lq, d), offsets, t, dtype)}
        if not s["train"]:
            return out
        do = _to_clouds(s["do"], offsets, lq).reshape(n, hk, h // hk * lq, d)
        dv = p.transpose(2, 3) @ do
        ds = (do @ v.transpose(2, 3)).sub_((do * o).sum(-1, keepdim=True)).mul_(p).mul_(scale)
        out["dq"] = _to_packed((ds @ k).reshape(n, h, lq, d), offsets, t, dtype)
        out["dk"] = _to_packed(ds.transpose(2, 3) @ q, offsets_k, tk, dtype)
        out["dv"] = _to_packed(dv, offsets_k, tk, dtype)
        return out


def _cached_plain(s):
    with torch.no_grad():
        (n, h, d), (_, p, hk, _) = s["q"].shape, s["k"].shape
        q = s["q"].float().reshape(n, hk, h // hk, d)
        k, v = s["k"].float().transpose(1, 2), s["v"].float().transpose(1, 2)
        hidden = torch.arange(p, device=DEVICE)[None, :] >= s["lengths"][:, None]
        w = ((q @ k.transpose(2, 3)) / math.sqrt(d)).masked_fill_(hidden[:, None, None], -math.inf)
        w = (w - w.amax(-1, keepdim=True)).exp()
        o = (w / w.sum(-1, keepdim=True)) @ v
        return {"o": o.reshape(n, h, d).to(s["q"].dtype)}


def _norm_own(s):
    import torch_point_ops_b200 as tpo

    y = tpo.layer_norm(s["x"], s["weight"], s["bias"], s["eps"])
    if not s["train"]:
        return {"y": y}
    dx, dw, db = torch.autograd.grad(y, (s["x"], s["weight"], s["bias"]), s["dy"])
    return {"y": y, "dx": dx, "dweight": dw, "dbias": db}


def _packed_own(s):
    import torch_point_ops_b200 as tpo

    o = tpo.packed_attention(s["q"], s["k"], s["v"], s["offsets"], s["offsets_k"], causal=s["case"]["causal"])
    if not s["train"]:
        return {"o": o}
    dq, dk, dv = torch.autograd.grad(o, (s["q"], s["k"], s["v"]), s["do"])
    return {"o": o, "dq": dq, "dk": dk, "dv": dv}


def _cached_own(s):
    import torch_point_ops_b200 as tpo

    return {"o": tpo.cached_attention(s["q"], s["k"], s["v"], s["lengths"])}


def run(state):
    plain, ours = {"norm": (_norm_plain, _norm_own), "packed": (_packed_plain, _packed_own),
                   "cached": (_cached_plain, _cached_own)}[state["case"]["op"]]
    return (ours if own else plain)(state)


def work(case):
    size = SIZE[case["dtype"]]
    if case["op"] == "norm":
        r, c = case["rows"], case["width"]
        if case["train"]:  # x and dy read, y and dx written; the weight, the bias and their gradients
            return {"bytes": 4 * r * c * size + 4 * c * size, "flops": 20 * r * c}
        return {"bytes": 2 * r * c * size + 2 * c * size, "flops": 8 * r * c}
    h, hk, d = case["heads"], case["kv_heads"], case["width"]
    lq, lk = _lengths(case)
    if case["op"] == "cached":
        return {"bytes": 2 * sum(lq) * hk * d * size + 2 * case["clouds"] * h * d * size,
                "flops": 4 * sum(lq) * h * d}
    pairs = sum(a * b - (a * (a - 1) // 2 if case["causal"] else 0) for a, b in zip(lq, lk))
    moved_q, moved_k = sum(lq) * h * d * size, sum(lk) * hk * d * size
    if case["train"]:  # q, do, k, v read, o, dq, dk, dv written; two products forward, five backward
        return {"bytes": 4 * moved_q + 4 * moved_k, "flops": 14 * pairs * h * d}
    return {"bytes": 2 * moved_q + 2 * moved_k, "flops": 4 * pairs * h * d}


def _attend_exact(q, k, v, hidden):
    """Rows q over keys k in 64 bits: probabilities and output; a row that sees nothing gives zeros."""
    score = (q @ k.mT) / math.sqrt(q.shape[-1])
    weight = torch.where(hidden, torch.zeros((), dtype=torch.float64, device=q.device),
                         torch.exp(score - score.masked_fill(hidden, -1e300).amax(-1, keepdim=True)))
    total = weight.sum(-1, keepdim=True)
    prob = weight / torch.where(total > 0, total, torch.ones_like(total))
    return prob, prob @ v


def exact(case, seed):
    s = prepare(case, seed)
    s = {k: v.detach().double() if isinstance(v, torch.Tensor) and v.is_floating_point() else v for k, v in s.items()}
    if case["op"] == "norm":
        x, w = s["x"], s["weight"]
        var, mean = torch.var_mean(x, 1, correction=0, keepdim=True)
        unit = (x - mean) / (var + s["eps"]).sqrt()
        out = {"y": unit * w + s["bias"]}
        if case["train"]:
            g, c = s["dy"] * w, case["width"]
            inner = (g * unit).sum(1, keepdim=True)
            out["dx"] = (c * g - g.sum(1, keepdim=True) - unit * inner) / (c * (var + s["eps"]).sqrt())
            out["dweight"], out["dbias"] = torch.einsum("rc,rc->c", s["dy"], unit), s["dy"].sum(0)
        return out
    group = case["heads"] // case["kv_heads"]
    lq, lk = _lengths(case)
    if case["op"] == "cached":
        o = torch.zeros_like(s["q"])
        for n, length in enumerate(lq):
            for head in range(case["kv_heads"]):
                rows = slice(head * group, (head + 1) * group)
                _, o[n, rows] = _attend_exact(s["q"][n, rows], s["k"][n, :length, head], s["v"][n, :length, head],
                                              torch.zeros(1, 1, dtype=torch.bool, device=DEVICE))
        return {"o": o}
    q, k, v = s["q"], s["k"], s["v"]
    out = {"o": torch.zeros_like(q)}
    if case["train"]:
        out.update(dq=torch.zeros_like(q), dk=torch.zeros_like(k), dv=torch.zeros_like(v))
    tq = tk = 0
    for a, b in zip(lq, lk):
        hidden = torch.zeros(a, b, dtype=torch.bool, device=DEVICE)
        if case["causal"]:
            hidden = torch.ones(a, b, dtype=torch.bool, device=DEVICE).triu(b - a + 1)
        rows, keys = slice(tq, tq + a), slice(tk, tk + b)
        for head in range(case["heads"]):
            kh = head // group
            prob, o = _attend_exact(q[rows, head], k[keys, kh], v[keys, kh], hidden)
            out["o"][rows, head] = o
            if case["train"]:
                g = s["do"][rows, head]
                out["dv"][keys, kh] += prob.mT @ g
                dp = g @ v[keys, kh].mT
                ds = prob * (dp - (prob * dp).sum(-1, keepdim=True)) / math.sqrt(case["width"])
                out["dq"][rows, head] = ds @ k[keys, kh]
                out["dk"][keys, kh] += ds.mT @ q[rows, head]
        tq, tk = tq + a, tk + b
    return out
