"""What the operators around a prompt, its scores and its continuations are measured on: three kinds of work.

  prompt   causal attention over dense rows of a prompt with grouped heads (``gemv.prompt_attention``): a batch, a padded batch
           behind a boolean mask, sequences of different lengths packed into one row axis, a few new rows behind many
           older ones (what the evaluation cache, which keeps values, is asked for at every step)
  score    log probabilities of given tokens from rows of logits, with the rows' entropy and their likeliest tokens
           (``gemv.token_logprobs``)
  take     sequences of a quantised cache copied over one another, moved to the front or forked, all layers' codes, checkpoints
           and states in one call (``gemv.take_sequences``): beams that go on from another one, finished sequences that leave
           a batch, one prompt that several answers begin with
"""
import math

import torch

own = False

DEV = "cuda:0"
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
INTERVAL = 256      # tokens between two recorded filter states of a cache
MOST_FLOPS, MOST_ROWS, MOST_LOGITS, MOST_CACHE = 2.1e12, 2.1e6, 1.4e8, 6e8     # of a drawn case: what the largest listed ones have


def _prompt(name, batch, kv_heads, group, tokens, rows=None, head_dim=128, dtype="fp16", padded=False, packed=0):
    """rows: the last ones of the tokens, which are asked (all of them); packed: that many sequences share the row axis."""
    return {"name": name, "kind": "prompt", "batch": batch, "kv_heads": kv_heads, "group": group, "tokens": tokens,
            "rows": tokens if rows is None else rows, "head_dim": head_dim, "dtype": dtype, "padded": padded, "packed": packed}


def _score(name, rows, vocab, top, dtype):
    return {"name": name, "kind": "score", "rows": rows, "vocab": vocab, "top": top, "dtype": dtype}


def _take(name, batch, rows, moved, kv_heads, tokens, layers, bits=4, fork=False):
    """moved: rows that another row takes the place of; fork: into new buffers, all rows."""
    return {"name": name, "kind": "take", "batch": batch, "rows": rows, "moved": moved, "kv_heads": kv_heads, "tokens": tokens,
            "layers": layers, "bits": bits, "fork": fork}


def listed():
    return [
        # one user's first message: launches and host calls count
        _prompt("prompt_short", 1, 32, 1, 160),
        # the prompts of the end-to-end generation benchmark's batch
        _prompt("prompt_batch", 128, 32, 1, 512),
        # a long document, grouped queries
        _prompt("prompt_long", 1, 8, 4, 16384, dtype="bf16"),
        # texts of different lengths, scored together without padding
        _prompt("prompt_packed", 1, 8, 4, 12001, dtype="bf16", packed=24),
        # a left-padded batch of prompts on a model with narrow heads
        _prompt("prompt_padded", 8, 16, 1, 1023, head_dim=64, padded=True),
        # a generated token in the evaluation model, which keeps dequantised values
        _prompt("prompt_step", 8, 8, 4, 4097, rows=1, dtype="bf16"),
        # a step of a beam search with four beams: two candidates for each
        _score("score_step", 4, 32000, 8, "fp32"),
        # a long prompt's own tokens
        _score("score_prompt", 4096, 32000, 0, "bf16"),
        # the likeliest alternatives of every token of a text, a large vocabulary of odd size
        _score("score_wide", 1000, 128001, 20, "fp16"),
        # the same search's cache: one of the four beams goes on as a second one, all layers
        _take("take_beams", 4, 4, 1, 32, 603, 32),
        # sequences that have ended leave a serving batch
        _take("take_leave", 64, 48, 12, 8, 4096, 4),
        # sixteen answers begin with one prompt and will go different ways, 2-bit codes
        _take("take_fork", 1, 16, 16, 8, 8001, 4, bits=2, fork=True),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["prompt", "prompt", "prompt", "score", "take"])
    while True:
        if kind == "prompt":
            kv, group = rng.choice([1, 2, 4, 5, 8, 16, 32]), rng.choice([1, 1, 2, 3, 4, 7, 8])
            tokens, form = _log(rng, 1, 16384), rng.choice(["batch", "batch", "padded", "packed", "rows"])
            c = _prompt("", 1 if form == "packed" else _log(rng, 1, 128), kv, group, tokens,
                        rows=_log(rng, 1, tokens) if form == "rows" else None, head_dim=rng.choice([64, 80, 96, 128, 128, 128, 256]),
                        dtype=rng.choice(["fp16", "bf16"]), padded=form == "padded", packed=_log(rng, 1, min(200, max(1, tokens // 4))) if form == "packed" else 0)
            if work(c)["flops"] <= MOST_FLOPS and c["batch"] * max(c["rows"] * group, tokens) * kv * c["head_dim"] <= MOST_ROWS * 128 \
                    and not (c["padded"] and c["batch"] * tokens * tokens > 1.4e8):
                break
        elif kind == "score":
            c = _score("", _log(rng, 1, 4096), _log(rng, 1000, 160000), rng.choice([0, 0, 1, 5, 8, 20, 32]), rng.choice(["fp16", "bf16", "fp32"]))
            if c["rows"] * c["vocab"] <= MOST_LOGITS:
                break
        else:
            fork = rng.random() < 0.3
            batch = _log(rng, 1 if fork else 2, 128)
            rows = _log(rng, batch, 128) if fork else rng.randint((batch + 1) // 2, batch)
            c = _take("", batch, rows, rows if fork else rng.randint(1, min(rows, batch - rows) if rows < batch else batch // 2),
                      rng.choice([1, 2, 5, 8, 32]), _log(rng, 1, 8192), _log(rng, 1, 32), rng.choice([4, 4, 2]), fork)
            if work(c)["bytes"] <= MOST_CACHE and batch * _row_bytes(c, True) <= 3 * MOST_CACHE:
                break
    del c["name"]
    return c


# ----------------------------------------------------------------------------------------------------- how much work
def _room(case):
    """Token slots of a cache that has grown to these tokens, and the slots per word."""
    per = 32 // case["bits"]
    return -(-int(case["tokens"] * 1.25) // 64) * 64, per


def _row_bytes(case, whole=False):
    """Of one sequence in all layers: codes, checkpoints and states of keys and values; whole: with what is still empty."""
    room, per = _room(case)
    words = (room if whole else -(-case["tokens"] // per) * per) // per
    marks = room // INTERVAL + 1 if whole else case["tokens"] // INTERVAL
    return 2 * case["layers"] * case["kv_heads"] * 128 * 4 * (words + marks + 1)


def work(case):
    if case["kind"] == "take":
        if case["fork"]:
            return {"bytes": case["batch"] * _row_bytes(case) + case["rows"] * _row_bytes(case, True), "flops": 0}
        return {"bytes": 2 * case["moved"] * _row_bytes(case), "flops": 0}
    if case["kind"] == "score":
        n, v, top = case["rows"], case["vocab"], case["top"]
        return {"bytes": n * v * DTYPES[case["dtype"]].itemsize + n * 16 + n * top * 12, "flops": 6 * n * v}
    b, h, g, t, r, d = (case[k] for k in ("batch", "kv_heads", "group", "tokens", "rows", "head_dim"))
    seen = r * (t - r) + r * (r + 1) / 2
    if case["packed"]:
        seen = sum(n * (n + 1) / 2 for n in _lengths(case))
    return {"bytes": 2 * d * (2 * b * h * t + 2 * b * h * g * r) + (b * t if case["padded"] else 0), "flops": 4 * d * b * h * g * seen}


def _lengths(case):
    """Of the packed sequences: long and short ones in turn, about as many of every order of size; they fill all rows but a few."""
    n, t = case["packed"], case["tokens"]
    share = [math.exp(3.0 * ((7 * i + 3) % n) / n) for i in range(n)]
    return [int(t * x / sum(share)) for x in share]


# ------------------------------------------------------------------------------------------------------ a user's data
def _prepare_prompt(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    b, h, g, t, r, d = (case[k] for k in ("batch", "kv_heads", "group", "tokens", "rows", "head_dim"))
    dt = DTYPES[case["dtype"]]
    rand = lambda *n: torch.randn(*n, generator=gen, device=DEV)
    # projections [B, T, heads, D] seen with the head axis first; some heads look around, some at few tokens
    made = lambda n, heads: (rand(b, n, heads, d) * torch.exp(0.5 * rand(heads, 1))).to(dt).transpose(1, 2)
    s = {"case": case, "q": made(r, h * g), "k": made(t, h), "v": rand(b, t, h, d).to(dt).transpose(1, 2), "mask": None, "bounds": None}
    if case["padded"]:      # true where a token is looked at, as attn_implementation="sdpa" has it; the first sequence is the longest
        pad = (torch.rand(b, generator=gen, device=DEV) * 0.7 * t).long()
        pad[0] = 0
        at = torch.arange(t, device=DEV)
        s["mask"] = ((at >= pad[:, None])[:, None, None, :] & (at[None, :] <= at[t - r:, None])).contiguous()
    if case["packed"]:
        lengths = _lengths(case)
        order = torch.randperm(len(lengths), generator=gen, device=DEV).cpu().tolist()
        ends = [0]
        for i in order:
            ends.append(ends[-1] + lengths[i])
        s["bounds"] = torch.tensor(ends, dtype=torch.int32, device=DEV)
    return s


def _prepare_score(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    n, v = case["rows"], case["vocab"]
    x = torch.randn(n, v, generator=gen, device=DEV).mul_(2.5)
    # a few likely tokens in every row, in some rows one that is nearly certain
    likely = torch.randint(0, v, (n, 6), generator=gen, device=DEV)
    x.scatter_add_(1, likely, 8.0 + 3.0 * torch.randn(n, 6, generator=gen, device=DEV))
    sure = torch.rand(n, 1, generator=gen, device=DEV) < 0.2
    x.scatter_add_(1, likely[:, :1], 14.0 * sure.float())
    other = torch.randint(0, v, (n,), generator=gen, device=DEV)
    tokens = torch.where(torch.rand(n, generator=gen, device=DEV) < 0.7, likely[:, 0], other)
    return {"case": case, "logits": x.to(DTYPES[case["dtype"]]), "tokens": tokens}


def _prepare_take(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    b, r, h, layers = (case[k] for k in ("batch", "rows", "kv_heads", "layers"))
    room, per = _room(case)
    words, marks = -(-case["tokens"] // per), case["tokens"] // INTERVAL
    # of all layers' keys and values, one after the other; a layer's are tensors of its own to the operator
    codes = torch.zeros(2 * layers, b, h, room // per, 128, dtype=torch.int32, device=DEV)
    ckpt = torch.zeros(2 * layers, b, h, room // INTERVAL + 1, 128, 2, dtype=torch.float16, device=DEV)
    state = torch.randn(2 * layers, b, h, 128, 2, generator=gen, device=DEV).half()
    for i in range(2 * layers):
        codes[i, :, :, :words] = torch.randint(-2 ** 31, 2 ** 31, (b, h, words, 128), generator=gen, device=DEV, dtype=torch.int32)
        ckpt[i, :, :, :marks] = torch.randn(b, h, marks, 128, 2, generator=gen, device=DEV).half()
    s = {"case": case, "whole": [codes, ckpt, state], "used": [words, marks, 128] * (2 * layers), "into": None}
    each = lambda whole: [t for layer in zip(*whole) for t in layer]
    s["tensors"] = each(s["whole"])
    if case["fork"]:
        index = torch.arange(r, device=DEV) % b
        s["whole"] = [torch.empty((2 * layers, r, *t.shape[2:]), dtype=t.dtype, device=DEV) for t in s["whole"]]
        s["into"] = each(s["whole"])
    else:
        # rows that go take the place of others, which are not asked for any more: those behind the rows that stay, or some that stay
        index = torch.arange(r, device=DEV)
        places = torch.randperm(r, generator=gen, device=DEV)
        sources = r + torch.randperm(b - r, generator=gen, device=DEV) if r < b else places[case["moved"]:]
        index[places[:case["moved"]]] = sources[:case["moved"]]
    s["index"] = index
    return s


def prepare(case, seed):
    return {"prompt": _prepare_prompt, "score": _prepare_score, "take": _prepare_take}[case["kind"]](case, seed)


# ------------------------------------------------------------------------------------------------------ one pass
def _pieces(s):
    """(sequence, its queries' rows, its keys' rows) of a call."""
    case = s["case"]
    if s["bounds"] is None:
        return [(i, slice(0, case["rows"]), slice(0, case["tokens"])) for i in range(case["batch"])]
    e = s["bounds"].tolist()
    return [(0, slice(x, y), slice(x, y)) for x, y in zip(e, e[1:])]


def _plain_prompt(s):
    case = s["case"]
    b, h, g, t, r, d = (case[k] for k in ("batch", "kv_heads", "group", "tokens", "rows", "head_dim"))
    out = torch.zeros(b, r, h * g, d, dtype=s["q"].dtype, device=DEV)
    most = max(1, int(1.1e9) // max(1, r * t * g))      # heads at a time
    for i, rows, seen in _pieces(s):
        n, m = rows.stop - rows.start, seen.stop - seen.start
        late = torch.arange(m, device=DEV) > torch.arange(m - n, m, device=DEV)[:, None]
        if s["mask"] is not None:
            late = late | ~s["mask"][i, 0]
        for h0 in range(0, h, most):
            heads = slice(h0, min(h, h0 + most))
            k, v = (s[x][i, heads, seen].float().contiguous() for x in ("k", "v"))
            q = s["q"][i, heads.start * g:heads.stop * g, rows].float().reshape(len(k), g * n, d)
            x = torch.bmm(q, k.transpose(1, 2).contiguous()).view(len(k), g, n, m).mul_(d ** -0.5).masked_fill_(late, -math.inf)
            top = x.amax(-1, keepdim=True) if m else x.new_zeros(len(k), g, n, 1)
            e = x.sub_(top.clamp_(min=-1e38)).exp_()
            total = e.sum(-1, keepdim=True)
            o = torch.bmm(e.view(len(k), g * n, m), v).view(len(k), g, n, d) / total
            o = torch.where(total > 0, o, 0.0)           # rows that look at nothing
            out[i, rows, heads.start * g:heads.stop * g] = o.reshape(len(k) * g, n, d).transpose(0, 1).to(out.dtype)
    return out


def _plain_score(s):
    case = s["case"]
    found = []
    for x, tokens in zip(s["logits"].split(512), s["tokens"].split(512)):
        d = x.double()                                   # long sums, and differences of nearly equal numbers
        d = d - d.amax(-1, keepdim=True)
        e = d.exp()
        total = e.sum(-1, keepdim=True)
        log = d - total.log()
        parts = [log.gather(1, tokens[:, None])[:, 0].float(), -(e * log).sum(-1).div(total[:, 0]).float()]
        if case["top"]:
            order = torch.sort(x, dim=-1, descending=True, stable=True)[1][:, :case["top"]].contiguous()
            parts += [log.gather(1, order).float(), order]
        found.append(parts)
    return [torch.cat(p) for p in zip(*found)]


def _plain_take(s):
    for t, to, used in zip(s["tensors"], s["into"] or s["tensors"], s["used"]):
        to[:len(s["index"]), :, :used] = t[s["index"], :, :used]
        if s["into"]:
            to[:, :, used:] = 0
    return s["whole"]


def run(s):
    kind = s["case"]["kind"]
    if not own:
        return {"prompt": _plain_prompt, "score": _plain_score, "take": _plain_take}[kind](s)
    from adkv_amd.kernel import gemv
    if kind == "prompt":
        return gemv.prompt_attention(s["q"], s["k"], s["v"], s["case"]["head_dim"] ** -0.5, s["mask"], bounds=s["bounds"])
    if kind == "score":
        r = gemv.token_logprobs(s["logits"], s["tokens"], top=s["case"]["top"])
        return list(r) if s["case"]["top"] else [r.logprobs, r.entropy]
    gemv.take_sequences(s["tensors"], s["index"], used=s["used"], into=s["into"])
    return s["whole"]


# ----------------------------------------------------------------------------------------- the definitions, in 64 bits
def _exact_prompt(case, seed):
    s = _prepare_prompt(case, seed)
    h, g, d = case["kv_heads"], case["group"], case["head_dim"]
    out = torch.zeros(case["batch"], case["rows"], h * g, d, dtype=torch.float64, device=DEV)
    at = torch.arange(case["tokens"], device=DEV)
    for i, rows, seen in _pieces(s):
        n, m = rows.stop - rows.start, seen.stop - seen.start
        for hq in range(h * g):
            k, v = s["k"][i, hq // g, seen].double(), s["v"][i, hq // g, seen].double()
            for r0 in range(0, n, 4096):
                r1 = min(n, r0 + 4096)
                to = m - n + r1                          # what the last of these rows looks at
                shown = at[:to] <= at[m - n + r0:to, None]
                if s["mask"] is not None:
                    shown = shown & s["mask"][i, 0, r0:r1, :to]
                x = torch.matmul(s["q"][i, hq, rows][r0:r1].double(), k[:to].t()) / math.sqrt(d)
                x[~shown] = -math.inf
                out[i, rows.start + r0:rows.start + r1, hq] = torch.matmul(torch.softmax(x, -1).nan_to_num_(0.0), v[:to])
    return out


def _exact_score(case, seed):
    s = _prepare_score(case, seed)
    found = []
    for x, tokens in zip(s["logits"].split(256), s["tokens"].split(256)):
        log = torch.log_softmax(x.double(), -1)
        parts = [log[torch.arange(len(x), device=DEV), tokens], torch.special.entr(log.exp()).sum(-1)]
        if case["top"]:
            parts += [log.sort(-1, descending=True)[0][:, :case["top"]], None]
        found.append(parts)
    return [None if p[0] is None else torch.cat(p) for p in zip(*found)]


def exact(case, seed):
    if case["kind"] == "take":
        return None
    return (_exact_prompt if case["kind"] == "prompt" else _exact_score)(case, seed)
