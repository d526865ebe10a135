"""The operators that score many positions of a text at once, each as a program calls it and as elementary tensor
operations:

  linear    a linear in 8-bit integers: a row of activations takes one scale (the row's largest magnitude / 127), a
            column of weights has its own, and out = (sum_k xq wq) * x_scale * w_scale
  logprobs  for each row of logits the log probability and the rank of a given token, the distribution's entropy and
            the most likely tokens
  attention rows of queries over the f16 cache, with scores capped by a tanh, a bias by distance, and a span of keys for
            each row: documents packed side by side, sliding windows, prompts that see themselves whole, a prefix that
            all documents share

Weights, activations, keys and values have the distributions of the synthetic models: int8 weights uniform with scales
that keep the products' size, activations, queries, keys and values N(0, 1), logits N(0, 2) with one likely token a row.
"""
import math

import torch

own = False  # True: run() calls the library's entries; False: the plain form

PAGE = 64       # positions per cache page (the paged configurations)
VOCAB = 151936  # the models' vocabulary
EPS = 1e-6


def listed():
    return [
        # q||k||v of the 27B shape for one token
        {"name": "linear_token", "kind": "linear", "rows": 1, "K": 5120, "N": 7168, "fp32": False},
        # gate||up over a ragged verification list
        {"name": "linear_verify13", "kind": "linear", "rows": 13, "K": 5120, "N": 34816, "fp32": False},
        # down over an ordinary, ragged prompt
        {"name": "linear_prompt_333", "kind": "linear", "rows": 333, "K": 17408, "N": 5120, "fp32": False},
        # gate||up over the largest chunk
        {"name": "linear_chunk_2048", "kind": "linear", "rows": 2048, "K": 5120, "N": 34816, "fp32": False},
        # the head over the positions of a text that is scored
        {"name": "linear_head_500", "kind": "linear", "rows": 500, "K": 5120, "N": VOCAB, "fp32": True},
        # a sampled token and its alternatives, token by token
        {"name": "logprobs_token", "kind": "logprobs", "rows": 1, "vocab": VOCAB, "used": VOCAB, "top": 20, "f16": False,
         "masked": 0},
        # an ordinary prompt: a padded vocabulary, logits rounded to f16 (ties)
        {"name": "logprobs_prompt_333", "kind": "logprobs", "rows": 333, "vocab": VOCAB, "used": 151669, "top": 5,
         "f16": True, "masked": 0},
        # the largest chunk of a scored text
        {"name": "logprobs_chunk_2048", "kind": "logprobs", "rows": 2048, "vocab": VOCAB, "used": VOCAB, "top": 20,
         "f16": False, "masked": 0},
        # one token of a sliding window layer with capped scores
        {"name": "attention_token_window", "kind": "attention", "q_heads": 40, "kv_heads": 8, "head_dim": 128, "rows": 1,
         "before": 4098, "window": 1024, "docs": 1, "shared": False, "given": 0, "cap": 50.0, "distance": False,
         "paged": False, "padded": 0},
        # one token at the far end of a long paged cache, capped scores
        {"name": "attention_token_128k", "kind": "attention", "q_heads": 40, "kv_heads": 8, "head_dim": 128, "rows": 1,
         "before": 131071, "window": 0, "docs": 1, "shared": False, "given": 0, "cap": 50.0, "distance": False,
         "paged": True, "padded": 0},
        # texts packed into one chunk, each seeing itself only, capped scores
        {"name": "attention_documents_2048", "kind": "attention", "q_heads": 40, "kv_heads": 8, "head_dim": 128,
         "rows": 2048, "before": 0, "window": 0, "docs": 7, "shared": False, "given": 0, "cap": 30.0, "distance": False,
         "paged": False, "padded": 0},
        # candidates behind a long prompt that they share, each with a part that sees itself whole, a bias by distance,
        # the chunk's last rows padding
        {"name": "attention_shared_777", "kind": "attention", "q_heads": 16, "kv_heads": 2, "head_dim": 256, "rows": 777,
         "before": 3001, "window": 0, "docs": 5, "shared": True, "given": 300, "cap": 0.0, "distance": True,
         "paged": True, "padded": 9},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["linear", "linear", "logprobs", "attention", "attention"])
    if kind == "linear":
        rows, K = _log_int(rng, 1, 2048), 64 * _log_int(rng, 4, 272)
        most = min(VOCAB, 2048 * 5120 * 34816 // (max(rows, 64) * K))
        return {"kind": kind, "rows": rows, "K": K, "N": 16 * _log_int(rng, 16, most // 16), "fp32": rng.random() < 0.4}
    if kind == "logprobs":
        used = _log_int(rng, 100, 200000)
        return {"kind": kind, "rows": _log_int(rng, 1, 2048 * 75000 // max(used, 75000)), "used": used,
                "vocab": used + rng.choice([0, 0, rng.randint(1, 300)]), "top": rng.choice([0, 1, 5, 20, 64]),
                "f16": rng.random() < 0.5, "masked": rng.choice([0, 0, 300])}
    c = {"kind": kind}
    c.update(rng.choice([{"q_heads": 40, "kv_heads": 8, "head_dim": 128}, {"q_heads": 32, "kv_heads": 8, "head_dim": 128},
                         {"q_heads": 16, "kv_heads": 16, "head_dim": 128}, {"q_heads": 16, "kv_heads": 2, "head_dim": 256},
                         {"q_heads": 24, "kv_heads": 4, "head_dim": 256}]))
    c["rows"] = rng.randint(1, 8) if rng.random() < 0.4 else _log_int(rng, 9, 2048)
    far = 65536 if c["rows"] <= 8 else min(8192, 2048 * 2048 // c["rows"])
    c["before"] = 0 if rng.random() < 0.25 else _log_int(rng, 1, far)
    c["window"] = _log_int(rng, 16, 4096) if rng.random() < 0.3 else 0
    c["docs"] = rng.randint(1, min(12, c["rows"])) if rng.random() < 0.6 else 1
    c["shared"] = c["docs"] > 1 and c["window"] == 0 and rng.random() < 0.6
    c["given"] = rng.choice([0, 0, 250, 600]) if c["window"] == 0 else 0
    c["cap"] = rng.choice([0.0, 30.0, 50.0])
    c["distance"] = rng.random() < 0.4
    c["paged"] = rng.random() < 0.5
    c["padded"] = rng.randint(0, c["rows"] // 3) if rng.random() < 0.3 else 0
    return c


# ---- inputs -------------------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal16(g, *shape, std=1.0):
    return torch.empty(shape, device="cuda", dtype=torch.float16).normal_(0.0, std, generator=g)


def _spans(c):
    """The rows' spans of keys, by the case alone: a row at cache position p sees the keys j < hi with j >= lo or
    j < prefix. Document d of the chunk begins at ragged fractions of it; the first `given` per mille of a document see
    each other whole; padding rows see nothing."""
    rows, before = c["rows"], c["before"]
    live = rows - c["padded"]
    cuts = sorted({int(live * math.modf(0.6180339887498949 * i)[0]) for i in range(1, c["docs"])} | {0})
    lo, hi = [], []
    for t in range(rows):
        start = max(x for x in cuts if x <= t)
        end = min([x for x in cuts if x > t] + [live])
        p = before + t
        a = 0 if c["docs"] == 1 else before + start
        if c["window"]:
            a = max(a, p + 1 - c["window"])
        lo.append(a)
        hi.append(0 if t >= live else max(p + 1, before + start + (end - start) * c["given"] // 1000))
    return lo, hi, before if c["shared"] else 0


def prepare(case, seed):
    c, g = dict(case), _gen(seed)
    s = {"c": c, "stream": torch.cuda.current_stream().cuda_stream}
    rows = c["rows"]
    if c["kind"] == "linear":
        K, N = c["K"], c["N"]
        s["x"] = _normal16(g, rows, K)
        s["w"] = torch.randint(-127, 128, (N, K), generator=g, device="cuda", dtype=torch.int8)
        # the library's layout of 8-bit weights, [N/16][K/64][k / 8 % 4][n % 16][k / 32 % 2][k % 8], laid out once
        s["tiled"] = s["w"].view(N // 16, 16, K // 64, 2, 4, 8).permute(0, 2, 4, 1, 3, 5).contiguous()
        s["scales"] = torch.empty(N, device="cuda").uniform_(0.5, 1.5, generator=g) / (73.0 * math.sqrt(K))
        s["out"] = torch.empty(rows, N, device="cuda", dtype=torch.float32 if c["fp32"] else torch.float16)
    elif c["kind"] == "logprobs":
        used = c["used"]
        x = torch.empty(rows, c["vocab"], device="cuda").normal_(0.0, 2.0, generator=g)
        likely = torch.randint(0, used, (rows,), generator=g, device="cuda")
        x.scatter_add_(1, likely[:, None], torch.empty(rows, 1, device="cuda").uniform_(0.0, 18.0, generator=g))
        if c["f16"]:
            x = x.half().float()
        if c["masked"]:  # a grammar that leaves some hundred tokens
            kept = torch.randint(0, used, (c["masked"],), generator=g, device="cuda")
            mask = torch.ones(c["vocab"], device="cuda", dtype=torch.bool)
            mask[kept] = False
            x.masked_fill_(mask, -math.inf)
        s["logits"] = x
        other = kept[torch.randint(0, len(kept), (rows,), generator=g, device="cuda")] if c["masked"] else \
            torch.randint(0, used, (rows,), generator=g, device="cuda")
        drawn = torch.where(torch.rand(rows, generator=g, device="cuda") < 0.5, likely, other)
        s["tokens"] = (other if c["masked"] else drawn).to(torch.int32)
        s["top"] = min(c["top"], used, 16 if c["masked"] and used < 1000 else 64)
        s["logprob"], s["entropy"] = (torch.empty(rows, device="cuda") for _ in range(2))
        s["rank"] = torch.empty(rows, device="cuda", dtype=torch.int32)
        s["ids"] = torch.empty(rows, s["top"], device="cuda", dtype=torch.int32)
        s["alternatives"] = torch.empty(rows, s["top"], device="cuda")
    else:
        qh, kvh, hd = c["q_heads"], c["kv_heads"], c["head_dim"]
        keys = c["before"] + rows
        n = -(-keys // PAGE) * PAGE
        s["q"] = torch.empty(rows, qh, hd, device="cuda").normal_(generator=g)
        s["k"], s["v"] = _normal16(g, kvh, n, hd), _normal16(g, kvh, n, hd)
        s["pages"] = torch.randperm(n // PAGE, generator=g, device="cuda", dtype=torch.int32) if c["paged"] else None
        lo, hi, s["prefix"] = _spans(c)
        s["lo"], s["hi"] = (torch.tensor(v, dtype=torch.int32, device="cuda") for v in (lo, hi))
        s["keys"], s["len"] = keys, n
        s["slopes"] = None
        if c["distance"]:  # 2^(-8 (h + 1) / heads)
            s["slopes"] = torch.exp2(-8.0 / qh * torch.arange(1, qh + 1, device="cuda", dtype=torch.float32))
        s["out"] = torch.empty(rows, qh, hd, device="cuda", dtype=torch.float16)
    return s


# ---- the library's entries ----------------------------------------------------------------------
def _p(t):
    return None if t is None else t.data_ptr()


def _bind(s):
    """The call of this state: a program fixes its buffers, sizes and workspace once and then repeats the call."""
    import importlib
    mi = importlib.import_module("intel-arc-inference-server_amd")
    c, st, L = s["c"], s["stream"], mi.lib()
    rows = c["rows"]

    def workspace(n):
        s["ws"] = torch.empty(max(n, 1), device="cuda", dtype=torch.uint8)
        return _p(s["ws"]), n

    if c["kind"] == "linear":
        K, N = c["K"], c["N"]
        args = ("mi_linear_w8a8", _p(s["x"]), K, _p(s["tiled"]), _p(s["scales"]),
                *workspace(L.mi_linear_w8a8_ws(rows, K)), _p(s["out"]),
                mi.OUT_F32 if c["fp32"] else mi.OUT_F16, N, rows, K, N, st)
        outs = s["out"]
    elif c["kind"] == "logprobs":
        args = ("mi_logprobs", _p(s["logits"]), c["vocab"], _p(s["tokens"]), rows, c["used"], s["top"], _p(s["logprob"]),
                _p(s["rank"]), _p(s["entropy"]), _p(s["ids"]) if s["top"] else None,
                _p(s["alternatives"]) if s["top"] else None, *workspace(L.mi_logprobs_ws(rows, c["used"], s["top"])), st)
        outs = _logprob_outputs(s["logprob"], s["rank"], s["entropy"], s["ids"], s["alternatives"])
    else:
        qh, kvh, hd, n = c["q_heads"], c["kv_heads"], c["head_dim"], s["len"]
        shape = mi.AttnShape(qh, kvh, hd, hd, 0, (qh + 2 * kvh) * hd, qh * hd, (qh + kvh) * hd, hd ** -0.5, EPS, 0)
        mask = mi.AttnMask(lo=_p(s["lo"]), hi=_p(s["hi"]), pos=None, pos0=c["before"], prefix=s["prefix"], cap=c["cap"],
                           slopes=_p(s["slopes"]))
        s["structs"] = shape, mask
        args = ("mi_attn_masked", _p(s["q"]), _p(s["k"]), _p(s["v"]), hd, n * hd, _p(s["pages"]), PAGE, n // PAGE,
                s["keys"], rows, mi.C.byref(shape), mi.C.byref(mask),
                *workspace(L.mi_attn_masked_ws(rows, s["keys"], mi.C.byref(shape))), _p(s["out"]), None, st)
        outs = s["out"]
    return mi.call, args, outs


# ---- one pass -----------------------------------------------------------------------------------
def _logprob_outputs(logprob, rank, entropy, ids, alternatives):
    return {"logprob": logprob, "rank": rank, "entropy": entropy, "ids": ids, "alternatives": alternatives}


def run(s):
    if own:
        if "call" not in s:
            s["call"] = _bind(s)
        call, args, outs = s["call"]
        call(*args)
        return outs
    return {"linear": _plain_linear, "logprobs": _plain_logprobs, "attention": _plain_attention}[s["c"]["kind"]](s)


def _plain_linear(s):
    x = s["x"].float()
    most = x.abs().amax(1, keepdim=True)
    scale = most / torch.full_like(most, 127.0)  # (by a Python number torch would multiply with its rounded inverse)
    q = torch.where(scale > 0, torch.round(x / scale), torch.zeros_like(x)).clamp(-127.0, 127.0)
    return ((q @ s["w"].float().t()) * scale * s["scales"]).to(s["out"].dtype)


def _plain_logprobs(s):
    used, top = s["c"]["used"], s["top"]
    x = s["logits"][:, :used] + 0.0  # (-0 counts as 0)
    at = s["tokens"].long()[:, None]
    d = x - x.amax(1, keepdim=True)
    e = d.exp()
    z = e.sum(1)
    log_z = z.log()
    entropy = log_z - torch.where(e > 0, e * d, torch.zeros_like(d)).sum(1) / z
    logprob = d.gather(1, at)[:, 0] - log_z
    # an integer key for each token in the order of rank: the larger logit, then the lower index
    bits = x.view(torch.int32)
    order = (bits ^ ((bits >> 31) & 0x7FFFFFFF)).long()
    key = (order << 32) + (0xFFFFFFFF - torch.arange(used, device=x.device))
    rank = (key > key.gather(1, at)).sum(1).to(torch.int32)
    ids = 0xFFFFFFFF - (key.topk(top, 1).values & 0xFFFFFFFF)
    return _logprob_outputs(logprob, rank, entropy, ids.to(torch.int32), d.gather(1, ids) - log_z[:, None])


def _rows_of_cache(s):
    j = torch.arange(s["keys"], device="cuda")
    return j if s["pages"] is None else s["pages"].long()[j // PAGE] * PAGE + j % PAGE


def _seen(s):
    j = torch.arange(s["keys"], device="cuda")
    lo, hi = s["lo"].long()[:, None], s["hi"].long()[:, None]
    return (j < hi) & ((j >= lo) | (j < s["prefix"]))


def _plain_attention(s):
    c = s["c"]
    qh, kvh, hd, rows, keys = c["q_heads"], c["kv_heads"], c["head_dim"], c["rows"], s["keys"]
    at = _rows_of_cache(s)
    k, v = s["k"][:, at].float(), s["v"][:, at].float()
    q = s["q"].view(rows, kvh, qh // kvh, hd).permute(1, 2, 0, 3).reshape(kvh, qh // kvh * rows, hd)
    w = (q @ k.transpose(1, 2).contiguous()) * hd ** -0.5
    if c["cap"]:
        w = c["cap"] * torch.tanh(w / c["cap"])
    w = w.view(qh, rows, keys)
    if c["distance"]:
        p = c["before"] + torch.arange(rows, device="cuda")
        far = (p[:, None] - torch.arange(keys, device="cuda")).abs().float()
        w = w - s["slopes"][:, None, None] * far
    w = torch.where(_seen(s), w, torch.full_like(w, -math.inf))
    m = w.amax(2, keepdim=True)
    e = torch.exp(w - torch.where(m == -math.inf, torch.zeros_like(m), m))
    z = e.sum(2, keepdim=True)
    o = (e.view(kvh, qh // kvh * rows, keys) @ v).view(qh, rows, hd) / torch.where(z > 0, z, torch.ones_like(z))
    return o.permute(1, 0, 2).to(torch.float16)


# ---- what a pass cannot do without --------------------------------------------------------------
def work(case):
    c = case
    rows = c["rows"]
    if c["kind"] == "linear":
        K, N = c["K"], c["N"]
        return {"bytes": 2 * rows * K + K * N + 4 * N + rows * N * (4 if c["fp32"] else 2), "flops": 2 * rows * K * N}
    if c["kind"] == "logprobs":
        n = rows * c["used"]
        return {"bytes": 4 * n + rows * (16 + 8 * c["top"]), "flops": 5 * n}
    lo, hi, prefix = _spans(c)
    pairs, first, last, shared = 0, None, 0, 0
    for a, b in zip(lo, hi):
        if b:
            part = min(prefix, a, b)  # keys of the prefix outside the span
            pairs += max(b - a, 0) + part
            first, last, shared = min(a, a if first is None else first), max(last, b), max(shared, part)
    keys = last - (first or 0) + min(shared, first or 0)
    qh, kvh, hd = c["q_heads"], c["kv_heads"], c["head_dim"]
    return {"bytes": rows * qh * hd * 6 + 4 * keys * kvh * hd, "flops": 4 * pairs * qh * hd}


# ---- the definitions in 64 bits -----------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return {"linear": _exact_linear, "logprobs": _exact_logprobs, "attention": _exact_attention}[case["kind"]](s)


def _exact_linear(s):
    # the scale is an fp32 number and the quotient an fp32 quotient (a quotient of two fp32 numbers formed in 64 bits
    # rounds to the fp32 one); the integers they give are exact, and so is everything after them
    x = s["x"].double()
    scale = (x.abs().max(dim=1).values / 127.0).float().double()
    q = torch.zeros_like(x)
    live = scale > 0
    q[live] = (x[live] / scale[live, None]).float().round().double().clamp(-127.0, 127.0)
    out = torch.empty(x.shape[0], s["w"].shape[0], device="cuda", dtype=torch.float64)
    step = 16384
    for n in range(0, out.shape[1], step):
        w = s["w"][n:n + step].double() * s["scales"][n:n + step, None].double()
        out[:, n:n + step] = (q @ w.t().contiguous()) * scale[:, None]
    return out


def _exact_logprobs(s):
    used, parts = s["c"]["used"], []
    for r in range(0, s["logits"].shape[0], 256):
        x = s["logits"][r:r + 256, :used].double()
        lse = torch.logsumexp(x, dim=1)
        lp = x - lse[:, None]
        p = lp.exp()
        entropy = -torch.nansum(p * lp, dim=1)  # (0 times -inf counts nothing)
        best = torch.sort(x, dim=1, descending=True, stable=True)
        ids = best.indices[:, :s["top"]]
        t = s["tokens"][r:r + 256].long()
        xt = x.gather(1, t[:, None])
        tied = (x == xt) & (torch.arange(used, device="cuda") < t[:, None])
        parts.append((lp.gather(1, t[:, None])[:, 0], ((x > xt) | tied).sum(1).to(torch.int32), entropy, ids.to(torch.int32),
                      lp.gather(1, ids)))
    return _logprob_outputs(*(torch.cat(v) for v in zip(*parts)))


def _exact_attention(s):
    c = s["c"]
    group, rows = c["q_heads"] // c["kv_heads"], c["rows"]
    at, seen = _rows_of_cache(s), _seen(s)
    empty = ~seen.any(1)
    far = (c["before"] + torch.arange(rows, device="cuda")[:, None] - torch.arange(s["keys"], device="cuda")).abs().double()
    out = torch.empty(rows, c["q_heads"], c["head_dim"], device="cuda", dtype=torch.float64)
    for h in range(c["q_heads"]):
        k, v = s["k"][h // group][at].double(), s["v"][h // group][at].double()
        w = torch.mm(s["q"][:, h].double(), k.t().contiguous()) / math.sqrt(c["head_dim"])
        if c["cap"]:
            w = torch.tanh(w / c["cap"]) * c["cap"]
        if c["distance"]:
            w -= float(s["slopes"][h]) * far
        w[~seen] = -math.inf
        w = torch.softmax(w, dim=1)
        w[empty] = 0.0
        out[:, h] = torch.mm(w, v)
    return out
