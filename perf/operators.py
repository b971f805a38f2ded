"""What the attention layer's operators around the quantised cache are measured on: two kinds of work.

  extend     n new tokens of every sequence: quantised, appended to the sequences' codes and attended with, over a prefix
             whose codes the batch shares and over each sequence's own codes (``gemv.extend``); n = 1 is a decode step
  rope_norm  the norm of every query and key head, its weight and the position rotation in one pass
             (``gemv.rope_norm_qk``); with ``train`` its gradients too

The codes are those of streams as the caches hold them: Gaussian rows, drifting outlier channels in the keys.
"""
import math

import torch

own = False

DEV = "cuda:0"
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
D = 128             # channels per head of a cache
INTERVAL = 256      # tokens between two recorded filter states
EPS = 1e-6
MOST_SCORES, MOST_FLOPS, MOST_OWN = 6.1e8, 3.1e11, 4.2e6   # of a drawn case: what the largest listed one has


def _extend(name, batch, kv_heads, group, prefix, tokens, new, bits=4, dtype="fp16", masked=False):
    return {"name": name, "kind": "extend", "batch": batch, "kv_heads": kv_heads, "group": group, "prefix": prefix, "tokens": tokens,
            "new": new, "bits": bits, "dtype": dtype, "masked": masked}


def _rope(name, batch, q_heads, kv_heads, tokens, head_dim, rotary, dtype="bf16", train=False):
    return {"name": name, "kind": "rope_norm", "batch": batch, "q_heads": q_heads, "kv_heads": kv_heads, "tokens": tokens,
            "head_dim": head_dim, "rotary": rotary, "dtype": dtype, "train": train}


def listed():
    return [
        # two requests that have just been sent on a short system prompt: their first generated token
        _extend("step_first", 2, 8, 4, 256, 0, 1),
        # the serving batch of the decode benchmark, all of it on one long system prompt, early in its answers
        _extend("step_wide", 128, 32, 1, 4096, 64, 1),
        # questions of different lengths about one document, left-padded, grouped queries, 2-bit codes
        _extend("step_masked_2bit", 48, 8, 4, 7777, 301, 1, bits=2, dtype="bf16", masked=True),
        # a few samples of one long prompt, well into their answers
        _extend("step_samples", 4, 32, 1, 8192, 1000, 1),
        # five drafted tokens per sequence are checked at once
        _extend("draft", 16, 8, 8, 2048, 200, 5, dtype="bf16"),
        # the questions themselves, left-padded, on top of the shared document: the largest call
        _extend("questions", 8, 32, 1, 4096, 0, 512, masked=True),
        # a follow-up turn in conversations that share nothing
        _extend("turn", 4, 8, 4, 0, 3001, 257, dtype="bf16"),
        # one generated token in the serving batch
        _rope("norm_step", 128, 32, 8, 1, 128, 128),
        # a prompt
        _rope("norm_prompt", 4, 32, 32, 2048, 128, 128, dtype="fp16"),
        # a training step of a long sequence, grouped queries
        _rope("norm_train", 2, 32, 8, 4096, 128, 128, train=True),
        # a small model in full precision, rotation of half of the channels
        _rope("norm_train_fp32", 3, 5, 5, 333, 64, 32, dtype="fp32", train=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    if rng.random() < 0.35:
        while True:
            dim = rng.choice([32, 64, 80, 96, 128, 128, 256])
            kv = rng.choice([1, 2, 4, 5, 8, 16, 32])
            c = _rope("", _log(rng, 1, 128), kv * rng.choice([1, 1, 2, 4, 8]), kv, _log(rng, 1, 4096), dim, rng.choice([dim, dim, dim // 2]),
                      dtype=rng.choice(["fp16", "bf16", "bf16", "fp32"]), train=rng.random() < 0.5)
            if c["batch"] * (c["q_heads"] + kv) * c["tokens"] * dim <= 4.2e7:
                del c["name"]
                return c
    while True:
        kv, group = rng.choice([1, 2, 4, 5, 8, 16, 32]), rng.choice([1, 1, 2, 4, 8])
        prefix = 0 if rng.random() < 0.15 else _log(rng, 1, 8192)
        tokens = 0 if rng.random() < 0.2 else _log(rng, 1, 3001)
        new = 1 if rng.random() < 0.5 else _log(rng, 2, 512)
        c = _extend("", _log(rng, 1, 128), kv, group, prefix, tokens, new, bits=rng.choice([4, 4, 2]), dtype=rng.choice(["fp16", "bf16"]),
                    masked=rng.random() < 0.4)
        b, seen = c["batch"], prefix + tokens + new
        if b * kv * group * new * seen <= MOST_SCORES and work(c)["flops"] <= MOST_FLOPS and b * kv * (tokens + new) <= MOST_OWN \
                and kv * prefix <= 262144:
            del c["name"]
            return c


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["kind"] == "rope_norm":
        b, t, d = case["batch"], case["tokens"], case["head_dim"]
        rows = b * t * (case["q_heads"] + case["kv_heads"])
        passes = 5 if case["train"] else 2        # read, write; read the rows and the gradient, write theirs
        return {"bytes": rows * d * size * passes + 2 * b * t * case["rotary"] * size * (2 if case["train"] else 1) + 4 * d * size,
                "flops": rows * d * (30 if case["train"] else 10)}
    b, h, g, p, t, n = (case[k] for k in ("batch", "kv_heads", "group", "prefix", "tokens", "new"))
    code = case["bits"] / 8
    seen = p + t + (n + 1) / 2
    rows = b * h * g * n
    byte = 2 * h * p * D * code + 2 * b * h * (t + n) * D * code + 2 * b * h * n * D * 2 + 2 * rows * D * 2
    return {"bytes": byte + (b * n * (p + t + n) * 2 if case["masked"] else 0),
            "flops": 4 * D * rows * seen + 6 * 2 * D * h * (p + b * (t + n))}


# --------------------------------------------------------------------------------------------- the streams' arithmetic
def _r16(x):
    """float64 to float16, rounded once: first to 24 bits with what is cut off kept in the last one, which float32 holds exactly."""
    b, m = x.view(torch.int64), (1 << 29) - 1
    return (((b & m) + m | b) & ~m).view(torch.float64).to(torch.float16)


def _fixed(params):
    """The parameters that do not change, [2, 1, H, D]: alpha, beta and 1 - beta * target, float64."""
    al, be, tg = (torch.stack([params[0][i], params[1][i]])[:, None] for i in (2, 3, 4))
    return al.double(), be.double(), (1.0 - be * tg).double()


def _advance(q, s, zp, sc, fixed):
    """The state after a code q of value s = r16(q * sc): r16(al * s + zp), r16(sc * r16(be * |q| + omt))."""
    al, be, omt = fixed
    return _r16(torch.addcmul(zp.double(), al, s.double())), sc * _r16(torch.addcmul(omt, be, q.abs().double()))


def _quantise(x, zp, sc, lo, hi):
    u = ((x.float() - zp.float()).double() / sc.double()).float()       # the IEEE quotient: 53 bits are enough to round twice
    return u.round_().clamp_(lo, hi).half()


def _range(bits):
    return -(1 << bits - 1), (1 << bits - 1) - 1


def _words(codes, bits):
    """Codes [2, X, H, T, D] as the cache's channel words [2, X, H, ceil(T / per), D], what is behind them zero."""
    two, x, h, t, d = codes.shape
    per = 32 // bits
    ns = -(-t // per)
    field = torch.zeros(two, x, h, ns * per, d, dtype=torch.int64, device=codes.device)
    field[:, :, :, :t] = codes.long() + (1 << bits - 1)
    shift = (bits * torch.arange(per, device=codes.device)).view(per, 1)
    return (field.view(two, x, h, ns, per, d) << shift).sum(4).to(torch.int32)


def _codes(words, bits, t):
    two, x, h, ns, d = words.shape
    shift = (bits * torch.arange(32 // bits, device=words.device, dtype=torch.int32)).view(-1, 1)
    field = (words[:, :, :, :, None] >> shift) & ((1 << bits) - 1)
    return (field.view(two, x, h, -1, d)[:, :, :, :t] - (1 << bits - 1)).half()


def _stream(rows, zp, sc, fixed, bits, first, record, value=None):
    """Quantises rows [n, 2, X, H, D] as the tokens from `first` on. Gives the codes like them and the state behind them;
    record(j, zp, sc) gets the state in front of token (j + 1) * INTERVAL."""
    lo, hi = _range(bits)
    codes = torch.empty(rows.shape, dtype=torch.float16, device=rows.device)
    for t in range(rows.shape[0]):
        q = _quantise(rows[t], zp, sc, lo, hi)
        s = q * sc
        codes[t] = q
        if value is not None:
            value[t] = s + zp
        zp, sc = _advance(q, s, zp, sc, fixed)
        if (first + t + 1) % INTERVAL == 0:
            record((first + t + 1) // INTERVAL - 1, zp, sc)
    return codes, zp, sc


def _replay(words, ckpt, start, fixed, bits, t):
    """The values of t tokens, [2, X, H, t, D], and the state behind them. The recorded states cut the stream into pieces that
    run side by side."""
    two, x, h, _, d = words.shape
    pieces = max(-(-t // INTERVAL), 1)
    last = t - (pieces - 1) * INTERVAL
    q = torch.zeros(two, x, h, pieces * INTERVAL, d, dtype=torch.float16, device=words.device)
    q[:, :, :, :t] = _codes(words, bits, t)
    q = q.view(two, x, h, pieces, INTERVAL, d).permute(4, 0, 1, 2, 3, 5).contiguous()
    zp, sc = (torch.cat([start[i].expand(two, x, h, d)[:, :, :, None], ckpt[:, :, :, :pieces - 1, :, i]], 3) for i in (0, 1))
    fixed = [f[:, :, :, None] for f in fixed]
    end = [zp[:, :, :, -1], sc[:, :, :, -1]]
    value = torch.empty_like(q)
    for i in range(INTERVAL if pieces > 1 else last):
        s = q[i] * sc
        value[i] = s + zp
        zp, sc = _advance(q[i], s, zp, sc, fixed)
        if i == last - 1:
            end = [zp[:, :, :, -1], sc[:, :, :, -1]]
    return value.permute(1, 2, 3, 4, 0, 5).reshape(two, x, h, pieces * INTERVAL, d)[:, :, :, :t], *end


# ----------------------------------------------------------------------------------------------------- a user's data
def _rows(gen, t0, t, x, h):
    """Key and value rows [t, 2, X, H, D]: Gaussian, four channels of every key head drift."""
    r = torch.randn(t, 2, x, h, D, generator=gen, device=DEV)
    at = torch.arange(t0, t0 + t, device=DEV, dtype=torch.float64)
    for k in range(4):
        r[:, 0, :, :, 32 * k] += (8.0 * torch.sin(0.01 * (k + 1) * at)).float().view(t, 1, 1)
    return r


def _params(gen, h, bits):
    u = lambda: (0.9 + 0.099 * torch.rand(h, D, generator=gen, device=DEV)).half()
    full = lambda v: torch.full((h, D), v, device=DEV, dtype=torch.float16)
    return [(full(0.0), u(), u(), full(0.02), full(_range(bits)[1] / 2)) for _ in range(2)]


def _cache(words):
    two, x, h, ns, d = words.shape
    return [words[i].contiguous().view(torch.uint8).view(x, h, ns, d // 4, 4, 4) for i in range(2)]


def _prepare_extend(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    b, h, g, p, t, n, bits = (case[k] for k in ("batch", "kv_heads", "group", "prefix", "tokens", "new", "bits"))
    dt = DTYPES[case["dtype"]]
    params = _params(gen, h, bits)
    fixed = _fixed(params)
    zp, sc = (torch.stack([params[0][i], params[1][i]])[:, None] for i in (0, 1))
    s = {"case": case, "params": params}

    def stream(rows, zp, sc, room):
        x, tokens = rows.shape[2], rows.shape[0]
        ckpt = torch.zeros(2, x, h, (tokens + room) // INTERVAL + 1, D, 2, dtype=torch.float16, device=DEV)

        def record(j, zp, sc):
            ckpt[:, :, :, j, :, 0], ckpt[:, :, :, j, :, 1] = zp, sc
        codes, zp, sc = _stream(rows, zp, sc, fixed, bits, 0, record)
        per = 32 // bits
        words = torch.zeros(2, x, h, -(-(tokens + room) // per), D, dtype=torch.int32, device=DEV)
        words[:, :, :, :-(-tokens // per)] = _words(codes.permute(1, 2, 3, 0, 4), bits)
        return _cache(words), [ckpt[0].clone(), ckpt[1].clone()], zp, sc
    if p:
        cache, ckpt, zp, sc = stream(_rows(gen, 0, p, 1, h).half(), zp, sc, 0)
        s["prefix"] = (*cache, p, *params, *ckpt)
    # the own streams go on from the state behind the prefix
    s["own_params"] = [(zp[i, 0].contiguous(), sc[i, 0].contiguous(), *params[i][2:]) for i in range(2)]
    zp, sc = (v.expand(2, b, h, D).contiguous() for v in (zp, sc))
    s["cache"], s["ckpt"], _, _ = stream(_rows(gen, p, t, b, h).half(), zp, sc, n)
    # a layer's projections: [B, n, heads, D], seen with the head axis first
    new = _rows(gen, p + t, n, b, h).to(dt)
    s["new"] = [new[:, i].transpose(0, 1).contiguous().transpose(1, 2) for i in range(2)]
    s["q"] = torch.randn(b, n, h * g, D, generator=gen, device=DEV).to(dt).transpose(1, 2)
    s["mask"] = None
    if case["masked"]:     # the prefix is whole; what is behind it is left-padded, the first sequence not at all
        pad = (torch.rand(b, generator=gen, device=DEV) * 0.5 * (t + n)).long()
        pad[0] = 0
        at = torch.arange(p + t + n, device=DEV)
        hidden = (at >= p) & (at < p + pad[:, None])
        late = at[None, :] > p + t + torch.arange(n, device=DEV)[:, None]
        s["mask"] = torch.zeros(b, 1, n, p + t + n, dtype=dt, device=DEV).masked_fill_(hidden[:, None, None, :] | late, torch.finfo(dt).min)
    return s


def _prepare_rope(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    b, hq, h, t, d, r = (case[k] for k in ("batch", "q_heads", "kv_heads", "tokens", "head_dim", "rotary"))
    dt = DTYPES[case["dtype"]]
    rand = lambda *n: torch.randn(*n, generator=gen, device=DEV)
    s = {"case": case}
    # projections [B, T, heads, D] seen with the head axis first; heads of different sizes, as their norm is there for
    for name, heads in (("q", hq), ("k", h)):
        s[name] = (rand(b, t, heads, d) * torch.exp(rand(heads, 1))).to(dt).transpose(1, 2)
        s["w" + name] = (1.0 + 0.1 * rand(d)).to(dt)
        s["g" + name] = rand(b, heads, t, d).to(dt) if case["train"] else None
    first = torch.randint(0, 100000, (b, 1), generator=gen, device=DEV) if t == 1 else torch.zeros(b, 1, device=DEV)
    angle = (first + torch.arange(t, device=DEV)).double()[:, :, None] * 10000.0 ** (-torch.arange(0, r, 2, device=DEV).double() / r)
    angle = torch.cat([angle, angle], -1)
    s["cos"], s["sin"] = torch.cos(angle).to(dt), torch.sin(angle).to(dt)
    if case["train"]:
        for name in ("q", "k", "wq", "wk"):
            s[name].requires_grad_()
    return s


def prepare(case, seed):
    return (_prepare_extend if case["kind"] == "extend" else _prepare_rope)(case, seed)


# ------------------------------------------------------------------------------------------------------- one pass
def _plain_extend(s):
    case = s["case"]
    b, h, g, p, t, n, bits = (case[k] for k in ("batch", "kv_heads", "group", "prefix", "tokens", "new", "bits"))
    fixed = _fixed(s["params"])
    both = lambda pair: torch.stack([v.view(torch.int32).view(*v.shape[:3], D) for v in pair])
    words, ckpt = both(s["cache"]), torch.stack(s["ckpt"])
    start = [torch.stack([s["own_params"][0][i], s["own_params"][1][i]])[:, None] for i in (0, 1)]
    past, zp, sc = _replay(words, ckpt, start, fixed, bits, t)

    # the new tokens: quantised one after the other, their codes put into the caches, their states recorded
    def record(j, zp, sc):
        for i in range(2):
            s["ckpt"][i][:, :, j, :, 0], s["ckpt"][i][:, :, j, :, 1] = zp[i], sc[i]
    value = torch.empty(n, 2, b, h, D, dtype=torch.float16, device=DEV)
    rows = torch.stack([x.permute(2, 0, 1, 3) for x in s["new"]], 1).half()
    codes, _, _ = _stream(rows, zp, sc, fixed, bits, t, record, value)
    per = 32 // bits
    sg = t // per
    behind = _codes(words[:, :, :, sg:], bits, (words.shape[3] - sg) * per)
    behind[:, :, :, t - sg * per:t - sg * per + n] = codes.permute(1, 2, 3, 0, 4)
    room = _words(behind, bits)                      # what is behind the new tokens stays as it was
    for i in range(2):
        s["cache"][i].view(torch.int32).view(b, h, -1, D)[:, :, sg:] = room[i]

    kv = torch.cat([past, value.permute(1, 2, 3, 0, 4)], 3).float()
    q = s["q"].float().reshape(b, h, g, n, D)
    own_q = q.reshape(b * h, g * n, D)
    scores = [torch.bmm(own_q, kv[0].reshape(b * h, t + n, D).transpose(1, 2).contiguous()).view(b, h, g, n, t + n)]
    if p:
        pre = both(s["prefix"][:2])
        zs = [torch.stack([s["params"][0][i], s["params"][1][i]])[:, None] for i in (0, 1)]
        shared = _replay(pre, torch.stack(s["prefix"][5:7]), zs, fixed, bits, p)[0][:, 0].float()
        pre_q = q.permute(1, 0, 2, 3, 4).reshape(h, b * g * n, D)
        scores.insert(0, torch.bmm(pre_q, shared[0].transpose(1, 2).contiguous()).view(h, b, g, n, p).transpose(0, 1))
    x = torch.cat(scores, -1) if p else scores[0]
    x = x * D ** -0.5
    if s["mask"] is not None:
        x = x + s["mask"].float()[:, :, None]
    late = torch.arange(p + t + n, device=DEV)[None, :] > p + t + torch.arange(n, device=DEV)[:, None]
    x = x.masked_fill(late, -math.inf)
    e = torch.exp(x - x.amax(-1, keepdim=True))
    w = e / e.sum(-1, keepdim=True)
    out = torch.bmm(w[..., p:].reshape(b * h, g * n, t + n), kv[1].reshape(b * h, t + n, D)).view(b, h, g, n, D)
    if p:
        out = out + torch.bmm(w[..., :p].transpose(0, 1).reshape(h, b * g * n, p), shared[1]).view(h, b, g, n, D).transpose(0, 1)
    return out.reshape(b, h * g, n, D).transpose(1, 2).contiguous().to(s["q"].dtype)


def _extended(s, out):
    return {"out": out, "k_cache": s["cache"][0], "v_cache": s["cache"][1], "k_ckpt": s["ckpt"][0], "v_ckpt": s["ckpt"][1]}


def _plain_rope(x, w, cos, sin):
    f = x.float()
    y = f * torch.rsqrt(f.square().mean(-1, keepdim=True) + EPS) * w.float()
    c, s = cos.float()[:, None], sin.float()[:, None]
    a, b, rest = y.split([c.shape[-1] // 2, c.shape[-1] // 2, y.shape[-1] - c.shape[-1]], -1)
    turned = torch.cat([a, b], -1) * c + torch.cat([-b, a], -1) * s
    return torch.cat([turned, rest], -1)


def _plain_rope_train(s):
    out = {}
    for n in ("q", "k"):
        x, w = s[n].detach().float().requires_grad_(), s["w" + n].detach().double().requires_grad_()
        rows = w.expand(*x.shape[:3], -1)            # the weight's gradient is a long sum: in 64 bits
        y = _plain_rope(x, rows, s["cos"], s["sin"])
        gx, gw = torch.autograd.grad(y, (x, w), s["g" + n].float())
        out |= {n: y.detach().to(s[n].dtype).contiguous(), "d" + n: gx.to(s[n].dtype).contiguous(), "dw" + n: gw.to(s["w" + n].dtype)}
    return out


def run(s):
    case = s["case"]
    if case["kind"] == "extend":
        if not own:
            return _extended(s, _plain_extend(s))
        from adkv_amd.kernel import gemv
        out = gemv.extend(s["q"], *s["cache"], *s["new"], *s["own_params"], case["tokens"], D ** -0.5, s["mask"],
                          prefix=gemv.SharedPrefix(*s["prefix"]) if "prefix" in s else None, k_ckpt=s["ckpt"][0], v_ckpt=s["ckpt"][1],
                          ckpt_interval=INTERVAL, bits=case["bits"])
        return _extended(s, out)
    if not own:
        if case["train"]:
            return _plain_rope_train(s)
        return {n: _plain_rope(s[n], s["w" + n], s["cos"], s["sin"]).to(s[n].dtype).contiguous() for n in ("q", "k")}
    from adkv_amd.kernel import gemv
    q, k = gemv.rope_norm_qk(s["q"], s["k"], s["cos"], s["sin"], s["wq"], s["wk"], EPS)
    if not case["train"]:
        return {"q": q, "k": k}
    dq, dk, dwq, dwk = torch.autograd.grad((q, k), (s["q"], s["k"], s["wq"], s["wk"]), (s["gq"], s["gk"]))
    return {"q": q.detach(), "dq": dq, "dwq": dwq, "k": k.detach(), "dk": dk, "dwk": dwk}


# --------------------------------------------------------------------------------------- the definitions, in 64 bits
def _half(x):
    """The float64 x rounded to the numbers that float16 has, as float64."""
    e = (torch.frexp(x)[1] - 11).clamp_(min=-24).long()
    power = lambda e: (e + 1023 << 52).view(torch.float64)
    return torch.round(x * power(-e)) * power(e)


def _exact_values(code, params, zp, sc):
    """code(t): token t's codes, or rows to quantise with the state; the values of every token, one after the other."""
    al, be, tg = (v.double() for v in params)
    omt = _half(1.0 - _half(be * tg))
    found, t = [], 0
    while (q := code(t, zp, sc)) is not None:
        s = _half(q * sc)
        found.append(_half(s + zp))
        zp, sc = _half(al * s + zp), _half(sc * _half(be * q.abs() + omt))
        t += 1
    return found, zp, sc


def _exact_extend(case, seed):
    s = _prepare_extend(case, seed)
    b, h, g, p, t, n, bits = (case[k] for k in ("batch", "kv_heads", "group", "prefix", "tokens", "new", "bits"))
    per, lo, hi = 32 // bits, *_range(bits)
    kv = []
    for i in range(2):
        zp, sc = s["params"][i][0].double(), s["params"][i][1].double()
        parts = []
        if p:
            w = s["prefix"][i].view(torch.int32).view(h, -1, D)
            code = lambda at, zp, sc: ((w[:, at // per] >> bits * (at % per) & (1 << bits) - 1) + lo).double() if at < p else None
            found, zp, sc = _exact_values(code, s["params"][i][2:], zp, sc)
            parts.append(torch.stack(found, 1).expand(b, h, p, D))
        v = s["cache"][i].view(torch.int32).view(b, h, -1, D)
        new = s["new"][i].half().double()

        def code(at, zp, sc):
            if at < t:
                return ((v[:, :, at // per] >> bits * (at % per) & (1 << bits) - 1) + lo).double()
            return torch.round(((new[:, :, at - t] - zp).float().double() / sc).float()).clamp_(lo, hi).double() if at < t + n else None
        found, _, _ = _exact_values(code, s["params"][i][2:], zp.expand(b, h, D), sc.expand(b, h, D))
        kv.append(torch.cat([*parts, torch.stack(found, 2)], 2))
    out = torch.empty(b, n, h * g, D, dtype=torch.float64, device=DEV)
    late = torch.arange(p + t + n, device=DEV)[None, :] > p + t + torch.arange(n, device=DEV)[:, None]
    for at in range(b):
        q = s["q"][at].double().view(h, g, n, D)
        x = torch.matmul(q, kv[0][at][:, None].transpose(2, 3)) * D ** -0.5
        if s["mask"] is not None:
            x = x + s["mask"][at].double()
        w = torch.softmax(x.masked_fill(late, -math.inf), -1)
        out[at] = torch.matmul(w, kv[1][at][:, None]).reshape(h * g, n, D).transpose(0, 1)
    return {"out": out, "k_cache": None, "v_cache": None, "k_ckpt": None, "v_ckpt": None}


def _exact_rope(case, seed):
    s = _prepare_rope(case, seed)
    d, r = case["head_dim"], case["rotary"]
    c, sn = (torch.nn.functional.pad(v.double(), (0, d - r), value=one)[:, None] for v, one in ((s["cos"], 1.0), (s["sin"], 0.0)))
    to = torch.arange(d, device=DEV)
    to[:r] = (to[:r] + r // 2) % r                   # channel i turns with channel to[i], which is its own partner's partner
    sign = torch.where(torch.arange(d, device=DEV) < r // 2, -1.0, 1.0).double()
    out = {}
    for n in ("q", "k"):
        x, w = s[n].detach().double(), s["w" + n].detach().double()
        rms = (x.pow(2).sum(-1, keepdim=True) / d + EPS).rsqrt()
        unit = x * rms
        y = unit * w
        out[n] = y * c + y[..., to] * sign * sn
        if case["train"]:
            gy = s["g" + n].double()
            back = gy * c + (gy * sn * sign)[..., to]
            gu = back * w
            out |= {"d" + n: rms * (gu - unit * (gu * unit).mean(-1, keepdim=True)), "dw" + n: (back * unit).sum((0, 1, 2))}
    return out


def exact(case, seed):
    return (_exact_extend if case["kind"] == "extend" else _exact_rope)(case, seed)
