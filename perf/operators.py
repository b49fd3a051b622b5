"""Operators of a sequence model over streams of path features (signatures of windows as tokens): what is measured of them.

Three operators ("op"), each in the forms a program calls:

  recurrence   h_t = exp(log_decay_t) h_{t-1} + x_t for each channel: forward, training step (forward and gradients), one
               token against a kept state
  rotary       norms of queries and keys for each head and the rotation by their positions, in one pass: forward, training
               step
  attention    causal attention with grouped heads over packed sequences of different lengths: forward, training step, one
               new token of each sequence against a cache

listed() holds fixed cases, draw() makes more of the same ranges.
"""
import math
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
TABLE = 32768               # positions that the rotation's tables hold
EPS = 1e-6


def _recurrence(name, mode, dtype, batch, length, channels, ragged=False):
    c = dict(op="recurrence", mode=mode, dtype=dtype, batch=batch, length=length, channels=channels, ragged=ragged)
    return dict(c, name=name) if name else c


def _rotary(name, mode, dtype, tokens, heads, kv_heads, dim, rotary, interleaved=False):
    c = dict(op="rotary", mode=mode, dtype=dtype, tokens=tokens, heads=heads, kv_heads=kv_heads, dim=dim, rotary=rotary,
             interleaved=interleaved)
    return dict(c, name=name) if name else c


def _attention(name, mode, dtype, batch, longest, shortest, past, heads, kv_heads, dim, causal=True):
    """`batch` sequences of `shortest` to `longest` queries each, and 0 to `past` keys before them."""
    c = dict(op="attention", mode=mode, dtype=dtype, batch=batch, longest=longest, shortest=shortest, past=past, heads=heads,
             kv_heads=kv_heads, dim=dim, causal=causal)
    return dict(c, name=name) if name else c


def listed():
    return [
        # online features: one new token of each of 64 streams against the states that are kept; nothing but latency
        _recurrence("recurrence_one_token", "step", "bf16", 64, 1, 2048),
        # an ordinary training step of a recurrent layer
        _recurrence("recurrence_train_bf16", "train", "bf16", 8, 2048, 2048),
        # one long recording in single precision, an odd number of samples
        _recurrence("recurrence_long_f32", "forward", "f32", 1, 100003, 384),
        # recordings of different lengths packed behind each other, an odd number of channels
        _recurrence("recurrence_packed_train_f16", "train", "f16", 37, 1500, 997, ragged=True),
        # the new tokens of 32 streams
        _rotary("rotary_one_token", "forward", "bf16", 32, 32, 8, 128, 128),
        # a long prompt
        _rotary("rotary_prompt_bf16", "forward", "bf16", 16384, 32, 8, 128, 128),
        # a training step in single precision, neighbouring channels of half of each head turned
        _rotary("rotary_train_f32", "train", "f32", 4099, 12, 4, 96, 48, interleaved=True),
        # one long prompt of a wide layer: the largest amount of arithmetic
        _attention("attention_prompt_bf16", "forward", "bf16", 1, 8192, 8192, 0, 32, 8, 128),
        # prompts of different lengths packed behind each other
        _attention("attention_packed_f16", "forward", "f16", 24, 2000, 1, 0, 16, 4, 64),
        # a training step of a wide layer over a few odd lengths
        _attention("attention_train_bf16", "train", "bf16", 4, 2047, 1600, 0, 32, 8, 128),
        # a training step over many short recordings, a window of a signature to a token
        _attention("attention_short_train_f16", "train", "f16", 200, 129, 17, 0, 8, 8, 64),
        # one new token of each of 48 streams against their caches
        _attention("attention_one_token", "forward", "bf16", 48, 1, 1, 12000, 32, 8, 128),
    ]


def _log(rng, low, high):
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49))))))


def draw(rng):
    op = rng.choice(["recurrence", "rotary", "attention"])
    if op == "recurrence":
        mode, dtype, channels = rng.choice(["forward", "train", "train", "step"]), rng.choice(list(DTYPES)), _log(rng, 16, 4096)
        if mode == "step":
            return _recurrence("", mode, dtype, _log(rng, 1, 256), 1, channels)
        batch = _log(rng, 1, 64)
        length = min(_log(rng, 16, 100000), max(1, 30000000 // (channels * batch)))
        return _recurrence("", mode, dtype, batch, length, channels, ragged=rng.random() < 0.4)
    if op == "rotary":
        mode, dtype = rng.choice(["forward", "train"]), rng.choice(list(DTYPES))
        dim, kv_heads = 8 * rng.randint(4, 16), rng.randint(1, 8)
        rotary = dim if rng.random() < 0.5 else 2 * rng.randint(1, dim // 2)
        heads = kv_heads * rng.randint(1, 8)
        tokens = min(_log(rng, 1, 16384), 80000000 // ((heads + kv_heads) * dim))
        return _rotary("", mode, dtype, tokens, heads, kv_heads, dim, rotary, interleaved=rng.random() < 0.5)
    mode, dtype = rng.choice(["forward", "train", "one_token"]), rng.choice(["bf16", "f16"])
    kv_heads, dim, batch = rng.randint(1, 8), rng.choice([64, 128, 64, 128, 32, 80, 96]), _log(rng, 1, 64)
    heads = kv_heads * rng.choice([1, 2, 3, 4, 6, 8])
    if mode == "one_token":
        past = min(_log(rng, 16, 32768), 150000000 // (batch * kv_heads * dim))
        return _attention("", "forward", dtype, batch, 1, 1, past, heads, kv_heads, dim)
    most = 1500000000 if mode == "forward" else 450000000          # scores of the plain form
    longest = max(16, min(_log(rng, 16, 8192), int(math.sqrt(most / (batch * heads)))))
    past = rng.choice([0, 0, longest // 2]) if mode == "forward" else 0
    return _attention("", mode, dtype, batch, longest, max(1, round(longest * rng.random())), past, heads, kv_heads, dim,
                      causal=rng.random() < 0.8)


def _lengths(case):
    """(queries, keys) of each sequence: they belong to the case, not to the seed."""
    rng = random.Random(1000 * case["batch"] + case.get("longest", case.get("length", 1)))
    if case["op"] == "recurrence":
        if not case["ragged"]:
            return [case["length"]] * case["batch"], None
        return [rng.randint(1, case["length"]) for _ in range(case["batch"])], None
    queries = [rng.randint(case["shortest"], case["longest"]) for _ in range(case["batch"])]
    queries[rng.randrange(case["batch"])] = case["longest"]
    past = [rng.randint(0, case["past"]) for _ in range(case["batch"])]
    past[rng.randrange(case["batch"])] = case["past"]
    return queries, [a + b for a, b in zip(queries, past)]


def _offsets(lengths):
    total, out = 0, [0]
    for n in lengths:
        total += n
        out.append(total)
    return out


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    dtype, op = DTYPES[case["dtype"]], case["op"]

    def normal(*shape, std=1.0, dtype=dtype):
        return (torch.randn(shape, generator=gen, device="cuda") * std).to(dtype)

    def whole(values):
        return torch.tensor(values, dtype=torch.int32, device="cuda")

    s = dict(case)
    if op == "recurrence":
        lengths, _ = _lengths(case)
        shape = (sum(lengths), case["channels"]) if case["ragged"] else (case["batch"], case["length"], case["channels"])
        # irregular sampling: a rate for each channel, from memories of one step to a thousand, times the time that passed
        rate = torch.exp(-6.9 * torch.rand(case["channels"], generator=gen, device="cuda"))
        passed = torch.empty((*shape[:-1], 1), device="cuda").exponential_(generator=gen)
        decay = -(rate * passed)
        s["log_decay"] = decay.to(dtype)
        s["x"] = (torch.randn(shape, generator=gen, device="cuda") * (-torch.expm1(2 * decay)).sqrt()).to(dtype)
        s["state"] = normal(case["batch"], case["channels"], dtype=torch.float32)
        s["steps"] = max(lengths)
        s["offsets"] = whole(_offsets(lengths))
        if case["mode"] == "step":
            s["log_decay"], s["x"] = s["log_decay"].squeeze(1), s["x"].squeeze(1)
        if case["mode"] == "train":
            s["grad"] = normal(*shape)
            s["grad_final"] = normal(case["batch"], case["channels"], dtype=torch.float32)
        return s
    if op == "rotary":
        tokens, heads, kv, dim = (case[k] for k in ("tokens", "heads", "kv_heads", "dim"))
        # queries and keys are parts of the output of one projection, the values behind them
        rows = normal(tokens, heads + 2 * kv, dim, std=1.3)
        s["q"], s["k"] = rows[:, :heads], rows[:, heads:heads + kv]
        s["q_weight"], s["k_weight"] = (1 + normal(dim, std=0.2, dtype=torch.float32) for _ in range(2))
        half = case["rotary"] // 2
        angle = torch.arange(TABLE, dtype=torch.float64, device="cuda")[:, None] * 10000.0 ** (
            -torch.arange(half, dtype=torch.float64, device="cuda") / half)
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
        if tokens <= 64:
            s["positions"] = torch.randint(0, TABLE, (tokens,), generator=gen, device="cuda", dtype=torch.int32)
        else:
            first = int(torch.randint(0, TABLE - tokens, (1,), generator=gen, device="cuda"))
            s["positions"] = torch.arange(first, first + tokens, dtype=torch.int32, device="cuda")
        if case["mode"] == "train":
            s["grad_q"], s["grad_k"] = normal(tokens, heads, dim), normal(tokens, kv, dim)
        return s
    queries, keys = _lengths(case)
    heads, kv, dim = case["heads"], case["kv_heads"], case["dim"]
    s["longest_q"], s["longest_k"] = max(queries), max(keys)
    s["q_offsets"] = whole(_offsets(queries))
    s["q"] = normal(sum(queries), heads, dim, std=1.4)
    if case["past"]:
        # a cache with room for the longest sequence in each place
        room = max(keys)
        s["k_offsets"], s["k_lengths"] = whole([i * room for i in range(case["batch"] + 1)]), whole(keys)
        total = room * case["batch"]
    else:
        s["k_offsets"], s["k_lengths"] = whole(_offsets(keys)), None
        total = sum(keys)
    s["k"], s["v"] = normal(total, kv, dim, std=1.4), normal(total, kv, dim)
    if case["mode"] == "train":
        s["grad"] = normal(sum(queries), heads, dim)
    return s


# ---- the plain forms: elementary torch operations in 32 bits, rounded once at the end ----

def _scan(a, b, longest):
    """b_t + a_t (b_{t-1} + a_{t-1} (...)) along the first axis, by doubling; a is zero where a sequence begins."""
    step = 1
    while step < longest:
        b = torch.cat((b[:step], b[step:] + a[step:] * b[:-step]))
        a = torch.cat((a[:step], a[step:] * a[:-step]))
        step *= 2
    return b


def _plain_recurrence(s):
    dtype, shape = s["x"].dtype, s["x"].shape
    if s["mode"] == "step":
        s["state"].mul_(torch.exp(s["log_decay"].float())).add_(s["x"].float())
        return s["state"].to(dtype), s["state"]
    channels = shape[-1]
    a, b = torch.exp(s["log_decay"].float()).reshape(-1, channels), s["x"].float().reshape(-1, channels)
    first, last = s["offsets"][:-1].long(), s["offsets"][1:].long() - 1
    inner = a.index_fill(0, first, 0.0)
    h = _scan(inner, b.index_add(0, first, a[first] * s["state"]), s["steps"])
    final = h[last]
    out = [h.to(dtype).reshape(shape), final]
    if s["mode"] == "train":
        # the same scan from the other end: the gradient of h_t is its own plus exp(log_decay_{t+1}) times the next one's
        own_grad = s["grad"].float().reshape(-1, channels).index_add(0, last, s["grad_final"])
        after = torch.cat((inner[1:], torch.zeros_like(inner[:1])))
        dh = _scan(after.flip(0), own_grad.flip(0), s["steps"]).flip(0)
        before = torch.cat((torch.zeros_like(h[:1]), h[:-1])).index_copy(0, first, s["state"])
        out += [dh.to(dtype).reshape(shape), (dh * a * before).to(dtype).reshape(shape), (dh * a)[first]]
    return out


def _turned(x, cos, sin, rotary, interleaved):
    """The first `rotary` channels of each head turned in pairs: neighbours, or one of each half."""
    if interleaved:
        a, b = x[..., 0:rotary:2], x[..., 1:rotary:2]
        y = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
    else:
        a, b = x[..., :rotary // 2], x[..., rotary // 2:rotary]
        y = torch.cat((a * cos - b * sin, a * sin + b * cos), -1)
    return torch.cat((y, x[..., rotary:]), -1)


def _plain_rotary(s):
    at = s["positions"].long()
    cos, sin = s["cos"][at][:, None], s["sin"][at][:, None]
    dtype, options, out, grads = s["q"].dtype, (s["rotary"], s["interleaved"]), [], []
    for name in ("q", "k"):
        x, w = s[name].float(), s[name + "_weight"]
        r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
        out.append(_turned(x * r * w, cos, sin, *options).to(dtype))
        if s["mode"] == "train":
            g = _turned(s["grad_" + name].float(), cos, -sin, *options)
            u = g * w
            grads.append(((u - x * (r * r * (u * x).mean(-1, keepdim=True))) * r).to(dtype))
            grads.append((g * x * r).sum((0, 1)))
    return out + grads


def _padded(x, starts, lengths, longest, kv):
    """Packed rows as (sequences, key heads, heads of each * rows, dim), in 32 bits; rows past a sequence's end are others'."""
    at = (starts[:, None] + torch.arange(longest, device=x.device)).clamp(max=x.shape[0] - 1)
    x = x[at].float()                                   # (sequences, rows, heads, dim)
    n, rows, heads, dim = x.shape
    return x.reshape(n, rows, kv, heads // kv, dim).permute(0, 2, 3, 1, 4).reshape(n, kv, heads // kv * rows, dim)


def _packed(x, starts, total, heads, rows):
    """The other way: (total, heads, ...)."""
    t = torch.arange(total, device=x.device)
    of = torch.searchsorted(starts, t, right=True) - 1
    n, kv = x.shape[:2]
    return x.reshape(n, heads, rows, *x.shape[3:])[of, :, t - starts[of]]


def _plain_attention(s):
    q, k, v = s["q"], s["k"], s["v"]
    heads, dim, kv, dtype = q.shape[1], q.shape[2], k.shape[1], q.dtype
    group, lq, lk, scale = heads // kv, s["longest_q"], s["longest_k"], 1.0 / math.sqrt(dim)
    q0, k0 = s["q_offsets"].long(), s["k_offsets"].long()
    nq, nk = q0[1:] - q0[:-1], (k0[1:] - k0[:-1] if s["k_lengths"] is None else s["k_lengths"].long())
    q0, k0 = q0[:-1], k0[:-1]
    Q, K, V = _padded(q, q0, nq, lq, kv), _padded(k, k0, nk, lk, kv), _padded(v, k0, nk, lk, kv)
    i, j = torch.arange(lq, device=q.device)[:, None], torch.arange(lk, device=q.device)
    seen = (j < nk[:, None, None]) & (i < nq[:, None, None])
    if s["causal"]:
        seen = seen & (j <= i + (nk - nq)[:, None, None])
    hidden = ~seen[:, None, None]                       # (sequences, 1, 1, rows, keys)
    shape5 = (len(nq), kv, group, lq, lk)
    p = torch.matmul(Q, K.transpose(2, 3).contiguous()).mul_(scale)
    p.view(shape5).masked_fill_(hidden, -math.inf)
    top = p.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    lse = top + torch.log(total)
    p.div_(torch.where(total == 0, torch.ones_like(total), total))
    O = torch.matmul(p, V)
    rows = (q0, q.shape[0], heads, lq)
    out = [_packed(O, *rows).to(dtype), _packed(lse, *rows).squeeze(-1)]
    if s["mode"] == "train":
        D = _padded(s["grad"], q0, nq, lq, kv)
        D.view(len(nq), kv, group, lq, dim).masked_fill_((i >= nq[:, None, None])[:, None, None], 0.0)
        ds = torch.matmul(D, V.transpose(2, 3).contiguous())
        ds.sub_((D * O).sum(-1, keepdim=True)).mul_(p).mul_(scale)
        dq = torch.matmul(ds, K)
        keys = (k0, k.shape[0], kv, lk)
        dk = torch.matmul(ds.transpose(2, 3).contiguous(), Q)
        dv = torch.matmul(p.transpose(2, 3).contiguous(), D)
        out += [_packed(dq, *rows).to(dtype), _packed(dk, *keys).to(dtype), _packed(dv, *keys).to(dtype)]
    return out


# ---- the framework's operators ----

def _own_recurrence(s):
    import pysiglib_amd as P
    if s["mode"] == "step":
        return P.linear_recurrence_step(s["x"], s["log_decay"], s["state"]), s["state"]
    offsets = s["offsets"] if s["ragged"] else None
    h, final = P.linear_recurrence(s["x"], s["log_decay"], initial_state=s["state"], offsets=offsets)
    if s["mode"] == "forward":
        return [h, final]
    return [h, final, *P.linear_recurrence_backprop(h, s["log_decay"], s["grad"], grad_final=s["grad_final"],
                                                    initial_state=s["state"], offsets=offsets)]


def _own_rotary(s):
    import pysiglib_amd as P
    args = (s["q"], s["k"], s["q_weight"], s["k_weight"], s["cos"], s["sin"], s["positions"])
    options = dict(eps=EPS, interleaved=s["interleaved"])
    q, k = P.norm_rotary(*args, **options)
    if s["mode"] == "forward":
        return [q, k]
    dq, dk, dqw, dkw = P.norm_rotary_backprop(s["grad_q"], s["grad_k"], *args, **options)
    return [q, k, dq, dqw, dk, dkw]


def _own_attention(s):
    import pysiglib_amd as P
    args = (s["q"], s["k"], s["v"])
    out, lse = P.attention(*args, s["q_offsets"], s["k_offsets"], k_lengths=s["k_lengths"], causal=s["causal"])
    if s["mode"] == "forward":
        return [out, lse]
    return [out, lse, *P.attention_backprop(s["grad"], *args, out, lse, s["q_offsets"], s["k_offsets"], causal=s["causal"])]


def run(s):
    if own:
        return {"recurrence": _own_recurrence, "rotary": _own_rotary, "attention": _own_attention}[s["op"]](s)
    return {"recurrence": _plain_recurrence, "rotary": _plain_rotary, "attention": _plain_attention}[s["op"]](s)


def work(case):
    c, size, train = case, SIZE[case["dtype"]], case["mode"] == "train"
    if c["op"] == "recurrence":
        cells, states = sum(_lengths(c)[0]) * c["channels"], 4 * c["batch"] * c["channels"]
        # forward: two in, one out; gradients: one more in, two more out (decays and outputs are at hand from the forward)
        return {"bytes": cells * size * (6 if train else 3) + states * (4 if train else 2), "flops": cells * (7 if train else 2)}
    if c["op"] == "rotary":
        cells = c["tokens"] * (c["heads"] + c["kv_heads"]) * c["dim"]
        return {"bytes": cells * size * (4 if train else 2) + c["tokens"] * (4 + 4 * c["rotary"]), "flops": cells * (20 if train else 7)}
    queries, keys = _lengths(c)
    pairs = 0
    for a, b in zip(queries, keys):
        pairs += a * b - a * (a - 1) // 2 if c["causal"] else a * b
    q, kv = sum(queries) * c["heads"] * c["dim"] * size, sum(keys) * c["kv_heads"] * c["dim"] * size
    lse = 4 * sum(queries) * c["heads"]
    # two products of a head's dimension for each pair forward, five more for the gradients
    return {"bytes": (4 * q + 4 * kv if train else 2 * q + 2 * kv) + lse, "flops": pairs * c["heads"] * c["dim"] * (14 if train else 4)}


# ---- the definitions in 64 bits ----

def _exact_recurrence(s):
    lengths, _ = _lengths(s)
    channels = s["channels"]
    a = s["log_decay"].double().reshape(-1, channels).exp()
    x = s["x"].double().reshape(-1, channels)
    start = _offsets(lengths)
    # all sequences side by side, padded in front of time by nothing and behind it by what is never read
    order = torch.zeros((max(lengths), len(lengths)), dtype=torch.long)
    for n, (t, k) in enumerate(zip(start, lengths)):
        order[:, n] = torch.clamp(torch.arange(max(lengths)), max=k - 1) + t
    order = order.cuda()
    ends = torch.tensor(lengths, device="cuda")
    h, state = torch.empty_like(x), s["state"].double().clone()
    for t in range(max(lengths)):
        row = order[t]
        moved = a[row] * state + x[row]
        state = torch.where((t < ends)[:, None], moved, state)
        h[row] = state
    if s["mode"] == "step":
        return state, state
    shape = s["x"].shape
    out = [h.reshape(shape), state]
    if s["mode"] == "train":
        g = s["grad"].double().reshape(-1, channels)
        dx, da, back = torch.empty_like(x), torch.empty_like(x), s["grad_final"].double().clone()
        for t in range(max(lengths) - 1, -1, -1):
            live = torch.nonzero(t < ends).squeeze(1)
            row = order[t][live]
            grad = g[row] + back[live]
            before = h[row - 1] if t else s["state"].double()[live]
            dx[row] = grad
            da[row] = grad * a[row] * before
            back[live] = grad * a[row]
        out += [dx.reshape(shape), da.reshape(shape), back]
    return out


def _exact_rotary(s):
    q, dim, half = s["q"], s["dim"], s["rotary"] // 2
    angle_c, angle_s = s["cos"].double()[s["positions"].long()], s["sin"].double()[s["positions"].long()]
    if s["interleaved"]:
        one = 2 * torch.arange(half, device=q.device)
        two = one + 1
    else:
        one = torch.arange(half, device=q.device)
        two = one + half
    out, grads = [], []
    for name in ("q", "k"):
        x = s[name].detach().double().requires_grad_(True)
        w = s[name + "_weight"].double().requires_grad_(True)
        with torch.enable_grad():
            y = x / torch.sqrt(x.pow(2).sum(-1, keepdim=True) / dim + EPS) * w
            c, d = angle_c[:, None], angle_s[:, None]
            z = y.index_copy(2, one, y[..., one] * c - y[..., two] * d).index_copy(2, two, y[..., two] * c + y[..., one] * d)
        out.append(z.detach())
        if s["mode"] == "train":
            grads += torch.autograd.grad(z, (x, w), s["grad_" + name].double())
    return out + grads


def _exact_attention(s):
    queries, keys = _lengths(s)
    heads, kv, dim = s["heads"], s["kv_heads"], s["dim"]
    group, start = heads // kv, _offsets(queries)
    place = [i * max(keys) for i in range(len(keys))] if s["past"] else _offsets(keys)
    train = s["mode"] == "train"
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.zeros(s["q"].shape[:2], dtype=torch.float64, device="cuda")
    dq, dk, dv = (torch.zeros(s[n].shape, dtype=torch.float64, device="cuda") for n in ("q", "k", "v")) if train else (None,) * 3
    for n, (a, b) in enumerate(zip(queries, keys)):
        rows, cols = slice(start[n], start[n] + a), slice(place[n], place[n] + b)
        hide = torch.ones((a, b), dtype=torch.bool, device="cuda").triu(1 + b - a) if s["causal"] else None
        for g in range(kv):
            own_heads = slice(g * group, (g + 1) * group)
            Q, K, V = s["q"][rows, own_heads].double(), s["k"][cols, g].double(), s["v"][cols, g].double()
            score = torch.tensordot(Q, K, ([2], [1])) / dim ** 0.5              # (queries, heads of the group, keys)
            if hide is not None:
                score.masked_fill_(hide[:, None], -math.inf)
            norm = torch.logsumexp(score, 2)
            weight = torch.exp(score - norm[..., None])
            del score
            out[rows, own_heads], lse[rows, own_heads] = torch.tensordot(weight, V, ([2], [0])), norm
            if train:
                G = s["grad"][rows, own_heads].double()
                dv[cols, g] = torch.tensordot(weight, G, ([0, 1], [0, 1]))
                into = torch.tensordot(G, V, ([2], [1]))
                into = weight * (into - (weight * into).sum(2, keepdim=True)) / dim ** 0.5
                dq[rows, own_heads] = torch.tensordot(into, K, ([2], [0]))
                dk[cols, g] = torch.tensordot(into, Q, ([0, 1], [0, 1]))
    return [out, lse, dq, dk, dv] if train else [out, lse]


def exact(case, seed):
    s = prepare(case, seed)
    # the recurrence goes step by step: three small launches for each
    if s["op"] == "recurrence" and s["steps"] * (2 if s["mode"] == "train" else 1) > 200000:
        return None
    return {"recurrence": _exact_recurrence, "rotary": _exact_rotary, "attention": _exact_attention}[s["op"]](s)
