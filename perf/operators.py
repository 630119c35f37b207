"""The operators of a text encoder over packed descriptions, as cases: attention over packed sequences (grouped heads, causal or
full, forward or forward + backward), the same with a learned relative position bias by buckets, the root-mean-square norm with the
residual's addition, and the global gradient norm with clipping (in place over a list of tensors, and inside the optimizer's step).

`run` computes them in plain torch operations, or, where `own` is set, through the framework's entry points."""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}


# ---- cases -------------------------------------------------------------------------------------------------------------------
def text_of(lens):
    return ",".join(str(int(n)) for n in lens)


def lens_of(text):
    return [int(n) for n in text.split(",")]


def ragged(count, low, high, step):
    """`count` lengths from low to high, the same ones every time: what a batch of descriptions looks like"""
    return [low + (i * step) % (high - low + 1) for i in range(count)]


def attention(lens, heads, kv_heads, dim, kind, causal, train, klens=None, buckets=0, far=0):
    return {"op": "attention", "lens": text_of(lens), "klens": text_of(klens or lens), "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "type": kind, "causal": causal, "train": train, "buckets": buckets, "far": far}


def listed():
    return [
        # evaluation of one batch of 16 descriptions of up to 30 tokens in the model's own 32 bits: the smallest call, latency
        dict(attention(ragged(16, 6, 30, 7), 4, 4, 64, "f32", False, False, buckets=32, far=128), name="bias_text_f32"),
        # a training step's batch of 64 descriptions of up to 126 tokens (the longest the dataset keeps), 32 bits, both directions
        dict(attention(ragged(64, 8, 126, 37), 8, 8, 32, "f32", False, True, buckets=32, far=128), name="bias_train_f32"),
        # dialogues and captions of a whole scene: hundreds of tokens, 16 bits, full attention with the bias and its gradient
        dict(attention(ragged(32, 61, 700, 211), 8, 8, 64, "bf16", False, True, buckets=32, far=128), name="bias_train_bf16"),
        # long packed texts, causal, one-sided buckets, grouped heads
        dict(attention([2048, 3999, 2571], 16, 4, 64, "bf16", True, True, buckets=32, far=128), name="bias_long_bf16"),
        # a prompt batch, causal, grouped heads, forward only
        dict(attention([2049, 1000, 517, 1777, 130, 2719], 32, 8, 128, "bf16", True, False), name="prompt_bf16"),
        # the same kind of batch in training
        dict(attention([2049, 1000, 517, 1777, 130, 2719], 16, 4, 128, "bf16", True, True), name="prompt_train_bf16"),
        # one long sequence of odd length, fp16, causal, training
        dict(attention([12289], 8, 2, 64, "f16", True, True), name="long_train_f16"),
        # one query token each against keys of very different lengths: few rows, a long axis
        dict(attention([1] * 16, 16, 4, 128, "bf16", False, False, klens=ragged(16, 500, 8100, 2719)), name="single_bf16"),
        # the norm between two blocks on the words of one batch (16 x 30 rows of the text encoder's width), 32 bits
        {"op": "norm", "rows": 480, "width": 256, "type": "f32", "train": True, "name": "norm_text_f32"},
        # ... and on long packed texts of a wide encoder, 16 bits with 32-bit weights
        {"op": "norm", "rows": 8190, "width": 4096, "type": "bf16", "train": True, "name": "norm_train_bf16"},
        # the optimizer step with clipping on as many tensors and values as this model has (about 8 million in 167 tensors)
        {"op": "step", "tensors": 167, "values": 8000000, "spread": 5, "name": "step_model"},
        # clipping in place of a list of gradients of mixed types
        {"op": "clip", "tensors": 48, "values": 60000000, "spread": 9, "name": "clip_mixed"},
    ]


def logspread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["attention", "attention", "attention", "bias", "bias", "norm", "step", "clip"])
    if op == "norm":
        width = logspread(rng, 64, 8192)
        rows = logspread(rng, 1, max(2, 30000000 // width))
        return {"op": "norm", "rows": rows, "width": width, "type": rng.choice(["f32", "bf16", "f16"]), "train": rng.random() < 0.7}
    if op in ("step", "clip"):
        return {"op": op, "tensors": logspread(rng, 1, 170 if op == "step" else 60), "values": logspread(rng, 20000, 30000000), "spread": rng.randrange(1, 1000)}
    dim = rng.choice([32, 64, 64, 128])
    kv = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 1, 2, 4]) if kv <= 4 else 1
    kind = rng.choice(["bf16", "bf16", "f16", "f32"])
    train = rng.random() < 0.6
    causal = rng.random() < 0.5
    count = logspread(rng, 1, 64)
    longest = logspread(rng, 20, max(24, int((24000 if kind != "f32" else 6000) / math.sqrt(count * kv * group) / (2 if train else 1))))
    lens = [max(1, int(longest * rng.uniform(0.1, 1.0))) for _ in range(count)]
    if op == "bias":
        return attention(lens, kv * group, kv, dim, kind, causal, train, buckets=rng.choice([16, 32, 64]), far=rng.choice([64, 128, 200]))
    if rng.random() < 0.3:  # few queries against many keys
        klens = lens
        lens = [rng.choice([1, 1, 2, 7, 16]) for _ in klens]
        return attention(lens, kv * group, kv, dim, kind, False, False, klens=klens)
    return attention(lens, kv * group, kv, dim, kind, causal, train)


# ---- inputs ------------------------------------------------------------------------------------------------------------------
def bucket_map(buckets, far, both):
    """bucket of every clipped distance key - query in -far .. far: half of the buckets (of each side) hold one distance each, the rest
    grow by a constant factor up to `far`. The borders are compared in whole numbers: n^m * e^t >= far^t * e^m."""
    per = buckets // 2 if both else buckets
    single = per // 2
    steps = per - single

    def side(n):
        if n < single:
            return n
        t = 0
        while t + 1 < steps and n ** steps * single ** (t + 1) >= far ** (t + 1) * single ** steps:
            t += 1
        return single + t

    if both:
        return [side(abs(d)) + (per if d > 0 else 0) for d in range(-far, far + 1)]
    return [side(max(-d, 0)) for d in range(-far, far + 1)]


def offsets(lens, dev):
    total, cu = 0, [0]
    for n in lens:
        total += n
        cu.append(total)
    return torch.tensor(cu, dtype=torch.int32, device=dev)


def sizes_of(case):
    """tensor sizes of a model: many small vectors, some matrices, together about `values`"""
    n, total = case["tensors"], case["values"]
    weights = [1.0 + ((i * 7919 + case["spread"] * 104729) % 1009) ** 2 / 50.0 * (1 if i % 3 == 0 else 0.002) for i in range(n)]
    whole = sum(weights)
    return [max(1, int(total * w / whole)) for w in weights]


def prepare(case, seed):
    dev = "cuda"
    g = torch.Generator(device=dev)
    g.manual_seed(int(seed))
    if case["op"] == "norm":
        dt, shape = TYPES[case["type"]], (case["rows"], case["width"])
        make = lambda s: (torch.randn(shape, generator=g, device=dev) * s).to(dt)  # noqa: E731
        return {"case": case, "x": make(1.0).requires_grad_(case["train"]), "r": make(1.5).requires_grad_(case["train"]),
                "w": (1 + 0.2 * torch.randn(shape[1], generator=g, device=dev)).requires_grad_(case["train"]), "dy": make(1.0), "dh": make(0.7)}
    if case["op"] in ("step", "clip"):
        sizes = sizes_of(case)
        grads = [torch.randn(n, generator=g, device=dev) * (0.01 + 0.002 * (i % 7)) for i, n in enumerate(sizes)]
        if case["op"] == "clip":
            fresh = [t.to((torch.float32, torch.bfloat16, torch.float32, torch.float16)[i % 4]) for i, t in enumerate(grads)]
            return {"case": case, "fresh": fresh, "grads": [torch.empty_like(t) for t in fresh], "max_norm": 1.0}
        at, idx = 0, []
        for n in sizes:
            idx.append(torch.arange(at, at + n, device=dev))
            at += (n + 15) // 16 * 16
        flat = torch.zeros(at, device=dev)
        params = [torch.randn(n, generator=g, device=dev) * 0.05 for n in sizes]
        idx = torch.cat(idx)
        flat[idx] = torch.cat(params)
        state = {"case": case, "grads": grads, "idx": idx, "p": flat, "m": torch.zeros_like(flat), "v": torch.zeros_like(flat), "step": 0,
                 "max_norm": 1.0, "lr": 1e-3, "decay": 1e-5, "betas": (0.9, 1 - 2.0 ** -10)}  # 1 - beta is exact in 32 bits
        if own:  # the optimizer that a training program keeps
            from instancerefer_amd.optim import FlatAdam
            leaves = [torch.nn.Parameter(t) for t in params]
            state["opt"] = FlatAdam(leaves, lr=state["lr"], betas=state["betas"], weight_decay=state["decay"])
            for leaf, grad in zip(leaves, grads):
                leaf.grad = grad
        return state
    dt = TYPES[case["type"]]
    lens, klens = lens_of(case["lens"]), lens_of(case["klens"])
    make = lambda n, h, s: (torch.randn(n, h, case["dim"], generator=g, device=dev) * s).to(dt)  # noqa: E731
    state = {"case": case, "q": make(sum(lens), case["heads"], 1.2), "k": make(sum(klens), case["kv_heads"], 1.2),
             "v": make(sum(klens), case["kv_heads"], 1.0), "cu": offsets(lens, dev), "cuk": offsets(klens, dev),
             "longest": max(lens), "longest_k": max(klens), "do": make(sum(lens), case["heads"], 1.0)}
    if case["buckets"]:
        both = not case["causal"]
        state["table"] = torch.randn(case["buckets"], case["heads"], generator=g, device=dev).to(dt)
        state["map"] = torch.tensor(bucket_map(case["buckets"], case["far"], both), dtype=torch.int32, device=dev)
    if case["train"]:
        for name in ("q", "k", "v", "table"):
            if name in state:
                state[name].requires_grad_(True)
    return state


# ---- the framework's operators -----------------------------------------------------------------------------------------------
def run_own(state):
    case = state["case"]
    if case["op"] == "norm":
        from instancerefer_amd.dense import rms_norm_residual
        y, h = rms_norm_residual(state["x"], state["r"], state["w"], eps=1e-6)
        if not case["train"]:
            return y, h
        dx, dr, dw = torch.autograd.grad((y, h), (state["x"], state["r"], state["w"]), (state["dy"], state["dh"]))
        return y.detach(), h.detach(), dx, dr, dw
    if case["op"] == "clip":
        from instancerefer_amd.optim import clip_grads_
        torch._foreach_copy_(state["grads"], state["fresh"])  # a backward pass leaves new gradients in place
        norm = clip_grads_(state["grads"], state["max_norm"])
        return [norm] + state["grads"]
    if case["op"] == "step":
        opt = state["opt"]
        norm = opt.backward_step(max_norm=state["max_norm"])
        return norm, opt.flat_p, opt.exp_avg, opt.exp_avg_sq
    from instancerefer_amd.attention import attention_packed
    extra = {"bias": state["table"], "buckets": state["map"]} if case["buckets"] else {}
    o = attention_packed(state["q"], state["k"], state["v"], state["cu"], state["cuk"], causal=case["causal"], **extra)
    if not case["train"]:
        return o
    leaves = [state["q"], state["k"], state["v"]] + ([state["table"]] if case["buckets"] else [])
    return (o.detach(),) + torch.autograd.grad(o, leaves, state["do"])


# ---- the plain form ----------------------------------------------------------------------------------------------------------
def padded(x, cu, longest):
    """(rows, heads, dim) packed -> (sequences, heads, longest, dim) in 32 bits with zeros behind each sequence, and the row of each place"""
    at = cu[:-1].long()[:, None] + torch.arange(longest, device=x.device)
    there = torch.arange(longest, device=x.device) < (cu[1:] - cu[:-1]).long()[:, None]
    rows = torch.where(there, at, torch.zeros_like(at))
    return (x[rows].float() * there[:, :, None, None]).permute(0, 2, 1, 3).contiguous(), there


def packed(x, there):
    return x.permute(0, 2, 1, 3)[there].contiguous()


def plain_attention(state):
    case = state["case"]
    dt, group = TYPES[case["type"]], case["heads"] // case["kv_heads"]
    q, in_q = padded(state["q"].detach(), state["cu"], state["longest"])
    k, in_k = padded(state["k"].detach(), state["cuk"], state["longest_k"])
    v, _ = padded(state["v"].detach(), state["cuk"], state["longest_k"])
    k, v = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
    scale = 1.0 / math.sqrt(case["dim"])
    s = torch.matmul(q * scale, k.transpose(2, 3).contiguous())
    i = torch.arange(q.shape[2], device=q.device)[:, None]
    j = torch.arange(k.shape[2], device=q.device)[None, :]
    if case["buckets"]:
        bucket = state["map"].long()[(j - i).clamp(-case["far"], case["far"]) + case["far"]]
        s = s + state["table"].detach().float()[bucket].permute(2, 0, 1)
    visible = in_k[:, None, None, :]
    if case["causal"]:
        more = ((state["cuk"][1:] - state["cuk"][:-1]) - (state["cu"][1:] - state["cu"][:-1])).long()
        visible = visible & (j <= i + more[:, None, None, None])
    s = s.masked_fill_(~visible, -math.inf)
    p = s.sub_(s.amax(3, keepdim=True)).exp_()
    p = p.div_(p.sum(3, keepdim=True))
    o = torch.matmul(p, v)
    if not case["train"]:
        return packed(o, in_q).to(dt)
    do, _ = padded(state["do"], state["cu"], state["longest"])
    dv = torch.matmul(p.transpose(2, 3), do)
    ds = torch.matmul(do, v.transpose(2, 3).contiguous())
    ds = ds.sub_((do * o).sum(3, keepdim=True)).mul_(p)
    dq = torch.matmul(ds, k) * scale
    dk = torch.matmul(ds.transpose(2, 3), q) * scale
    fold = lambda t: t.reshape(t.shape[0], case["kv_heads"], group, t.shape[2], t.shape[3]).sum(2)  # noqa: E731
    got = (packed(o, in_q).to(dt), packed(dq, in_q).to(dt), packed(fold(dk), in_k).to(dt), packed(fold(dv), in_k).to(dt))
    if case["buckets"]:
        by_pair = ds.sum(0).flip(1)
        heads, lq, lk = by_pair.shape
        # row i moved right by lq - 1 - i places: column c then holds distance j - i = c - (lq - 1), so a sum down the rows is by distance
        moved = torch.nn.functional.pad(by_pair, (0, lq)).reshape(heads, -1)[:, : lq * (lk + lq - 1)].reshape(heads, lq, lk + lq - 1)
        by_distance = moved.sum(1, dtype=torch.float64)
        distance = torch.arange(-(lq - 1), lk, device=q.device)
        which = state["map"].long()[distance.clamp(-case["far"], case["far"]) + case["far"]]
        chosen = (which[:, None] == torch.arange(case["buckets"], device=q.device)).double()
        got += (torch.matmul(by_distance, chosen).t().contiguous().to(dt),)
    return got


def plain_norm(state):
    case = state["case"]
    dt = TYPES[case["type"]]
    h = (state["x"].detach().float() + state["r"].detach().float()).to(dt)  # what the residual stream holds
    f, w = h.float(), state["w"].detach()
    rstd = torch.rsqrt(f.square().mean(1, keepdim=True) + 1e-6)
    hat = f * rstd
    y = (hat * w).to(dt)
    if not case["train"]:
        return y, h
    dy = state["dy"].float()
    g = dy * w
    dh = state["dh"].float() + rstd * (g - hat * (g * hat).mean(1, keepdim=True))
    dw = (dy * hat).sum(0, dtype=torch.float64).float()
    return y, h, dh.to(dt), dh.to(dt), dw


def plain_clip(state):
    torch._foreach_copy_(state["grads"], state["fresh"])
    grads = state["grads"]
    total = torch.stack([g.float().square().sum(dtype=torch.float64) for g in grads]).sum()
    norm = total.sqrt()
    factor = (state["max_norm"] / (norm + 1e-6)).clamp(max=1.0).float()
    for g in grads:
        g.copy_(g.float() * factor)
    return [norm.float()] + grads


def plain_step(state):
    grad = torch.zeros_like(state["p"])
    grad[state["idx"]] = torch.cat(state["grads"])
    norm = grad.square().sum(dtype=torch.float64).sqrt()
    factor = (state["max_norm"] / (norm + 1e-6)).clamp(max=1.0).float()
    state["step"] += 1
    p, m, v = state["p"], state["m"], state["v"]
    grad = grad * factor + state["decay"] * p
    first, second = state["betas"]
    m.mul_(first).add_(grad * (1 - first))
    v.mul_(second).add_(grad * grad * (1 - second))
    step_size = state["lr"] / (1 - first ** state["step"])
    p.sub_(step_size * (m / (v.sqrt() / math.sqrt(1 - second ** state["step"]) + 1e-8)))
    return norm.float(), p, m, v


def run(state):
    if own:
        return run_own(state)
    return {"attention": plain_attention, "norm": plain_norm, "clip": plain_clip, "step": plain_step}[state["case"]["op"]](state)


# ---- what a pass cannot do without -------------------------------------------------------------------------------------------
def visible_pairs(lq, lk, causal):
    if not causal:
        return lq * lk
    return sum(max(0, min(lk, i + 1 + lk - lq)) for i in range(lq))


def work(case):
    if case["op"] == "norm":
        n, b = case["rows"] * case["width"], BYTES[case["type"]]
        passes = 4 + (4 if case["train"] else 0)  # x, r, y, h; dy, dh and the two (equal) gradients
        return {"bytes": n * b * passes + case["width"] * 8, "flops": n * (14 if case["train"] else 5)}
    if case["op"] == "clip":
        sizes = sizes_of(case)
        b = sum(n * (4, 2, 4, 2)[i % 4] for i, n in enumerate(sizes))
        return {"bytes": 4 * b, "flops": 3 * sum(sizes)}  # the copy, and read + write of the clipping
    if case["op"] == "step":
        n = sum(sizes_of(case))
        return {"bytes": 28 * n, "flops": 16 * n}
    lens, klens, b = lens_of(case["lens"]), lens_of(case["klens"]), BYTES[case["type"]]
    pairs = sum(visible_pairs(x, y, case["causal"]) for x, y in zip(lens, klens))
    rows, keys = sum(lens) * case["heads"] * case["dim"], sum(klens) * case["kv_heads"] * case["dim"]
    if case["train"]:  # q, do, o, dq and k, v, dk, dv
        return {"bytes": (4 * rows + 4 * keys) * b, "flops": 14.0 * pairs * case["heads"] * case["dim"]}
    return {"bytes": (2 * rows + 2 * keys) * b, "flops": 4.0 * pairs * case["heads"] * case["dim"]}


# ---- the definition in 64 bits -----------------------------------------------------------------------------------------------
def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "norm":
        x, r = state["x"].detach(), state["r"].detach()
        h = (x.double() + r.double()).to(x.dtype).double().requires_grad_(True)  # the stored sum is what the norm reads
        w = state["w"].detach().double().requires_grad_(True)
        y = w * h / torch.sqrt(torch.mean(h * h, dim=1, keepdim=True) + 1e-6)
        if not case["train"]:
            return y.detach(), h.detach()
        dh, dw = torch.autograd.grad(y, (h, w), state["dy"].double())
        dh = dh + state["dh"].double()
        return y.detach(), h.detach(), dh, dh, dw
    if case["op"] in ("clip", "step"):
        grads = [g.double() for g in state["fresh" if case["op"] == "clip" else "grads"]]
        norm = math.sqrt(sum(float(torch.dot(g, g)) for g in grads))
        factor = min(1.0, state["max_norm"] / (norm + 1e-6))
        if case["op"] == "clip":
            return [torch.tensor(norm, dtype=torch.float64)] + [g * factor for g in grads]
        p = state["p"].double()
        grad = torch.zeros_like(p)
        grad.index_copy_(0, state["idx"], torch.cat(grads) * factor)
        grad = grad + state["decay"] * p
        b1, b2 = state["betas"]
        m, v = (1 - b1) * grad, (1 - b2) * grad * grad
        p = p - state["lr"] * (m / (1 - b1)) / (torch.sqrt(v / (1 - b2)) + 1e-8)
        return torch.tensor(norm, dtype=torch.float64), p, m, v
    heads, per, dim = case["heads"], case["heads"] // case["kv_heads"], case["dim"]
    cu, cuk = state["cu"].tolist(), state["cuk"].tolist()
    out = {n: torch.zeros(state[n].shape, dtype=torch.float64, device="cuda") for n in ("q", "k", "v", "do")}
    dtable = torch.zeros((heads, max(1, case["buckets"])), dtype=torch.float64, device="cuda")
    for b in range(len(cu) - 1):
        rows, keys = slice(cu[b], cu[b + 1]), slice(cuk[b], cuk[b + 1])
        lq, lk = cu[b + 1] - cu[b], cuk[b + 1] - cuk[b]
        place = torch.arange(lq, device="cuda")[:, None] + (lk - lq) - torch.arange(lk, device="cuda")[None, :]  # query behind key by so much
        for h in range(heads):
            q = state["q"].detach()[rows, h].double()
            k, v = (state[n].detach()[keys, h // per].double() for n in ("k", "v"))
            score = (q @ k.t()) / math.sqrt(dim)
            if case["buckets"]:
                kind = state["map"].long()[case["far"] - place.clamp(-case["far"], case["far"])]
                score = score + state["table"].detach()[:, h].double()[kind]
            if case["causal"]:
                score = torch.where(place >= 0, score, torch.full_like(score, -math.inf))
            p = torch.exp(score - torch.logsumexp(score, 1, keepdim=True))
            del score
            o = p @ v
            out["do"][rows, h] = o
            if case["train"]:
                do = state["do"][rows, h].double()
                out["v"][keys, h // per] += p.t() @ do
                p = p * (do @ v.t() - (do * o).sum(1, keepdim=True))
                out["q"][rows, h] = p @ k / math.sqrt(dim)
                out["k"][keys, h // per] += p.t() @ q / math.sqrt(dim)
                if case["buckets"]:
                    for n in range(case["buckets"]):
                        dtable[h, n] += p[kind == n].sum()
    if not case["train"]:
        return out["do"]
    return (out["do"], out["q"], out["k"], out["v"]) + ((dtable.t().contiguous(),) if case["buckets"] else ())
