"""The operators of one decoding step of several sequences over a paged cache, with drafted trees or beams, each as a
program calls it and as elementary tensor operations:

  plan     block tables and slot maps from the requests' lengths: pages taken from and given back to a ring of free pages,
           each row's sequence, cache row and position, and the ancestors of each node of a tree
  table    the rotation's cosines and sines, with frequencies scaled for long contexts
  rotate   rows of q||k||v: norm of each head, rotation at the rows' own positions, q in 32 bits, k and v into cache rows
  tree     attention of every sequence's rows over its own pages: all cached keys, and of the step's own the ancestors
  select   the best continuations over beams and vocabulary
  move     rows of the cache to other rows, in every layer and head

Activations, keys and values are N(0, 1), norm weights N(1, 0.02), logits N(0, 2) with one likely token a row.
"""
import math

import torch

own = False  # True: run() calls the library's entries; False: the plain form

VOCAB = 151936  # the models' vocabulary
EPS = 1e-6
HEADS = [(40, 8, 128), (16, 2, 256), (32, 8, 128), (16, 16, 128), (24, 4, 256)]


def listed():
    return [
        # the next step of a few requests, each with a tree of drafts
        {"name": "plan_trees_8", "kind": "plan", "requests": 8, "rows": 61, "prompts": 0, "far": 4100, "page": 64, "tree": True},
        # a busy server: many single tokens, some prompts among them, some requests done
        {"name": "plan_requests_509", "kind": "plan", "requests": 509, "rows": 1, "prompts": 9, "far": 8000, "page": 16,
         "tree": False},
        # the rotation of a long context, made once for a run
        {"name": "table_131072", "kind": "table", "from": 0, "positions": 131072, "rot": 128, "scaling": "yarn", "factor": 4.0},
        # one token of a model that rotates a part of its heads in pairs of neighbours
        {"name": "rotate_token", "kind": "rotate", "heads": 1, "rows": 1, "rot": 64, "paired": True, "f16": True, "norm": True,
         "padded": 0},
        # the largest chunk of the 27B shape
        {"name": "rotate_chunk_2048", "kind": "rotate", "heads": 0, "rows": 2048, "rot": 128, "paired": False, "f16": False,
         "norm": True, "padded": 0},
        # one token of one sequence, where latency counts
        {"name": "tree_token_4098", "kind": "tree", "heads": 0, "sequences": 1, "rows": 1, "near": 4097, "far": 4097, "page": 64,
         "tree": False},
        # a batch of ragged sequences, a token each
        {"name": "tree_batch_48", "kind": "tree", "heads": 0, "sequences": 48, "rows": 1, "near": 130, "far": 16000, "page": 16,
         "tree": False},
        # a batch of sequences, each with a tree of drafts
        {"name": "tree_drafts_8", "kind": "tree", "heads": 0, "sequences": 8, "rows": 61, "near": 700, "far": 8200, "page": 64,
         "tree": True},
        # one tree at the far end of a long cache
        {"name": "tree_drafts_128k", "kind": "tree", "heads": 1, "sequences": 1, "rows": 60, "near": 131071, "far": 131071,
         "page": 64, "tree": True},
        # one text's beams
        {"name": "select_4", "kind": "select", "batch": 1, "beams": 4, "k": 8, "used": VOCAB, "done": False},
        # a batch's beams, some of them at their end
        {"name": "select_16x8", "kind": "select", "batch": 16, "beams": 8, "k": 16, "used": 151669, "done": True},
        # beams that go on from others: the page that each was writing is copied into one of its own
        {"name": "move_beams_32", "kind": "move", "layers": 40, "heads": 1, "lists": 32, "page": 64},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["plan", "table", "rotate", "tree", "tree", "tree", "select", "move"])
    if kind == "plan":
        tree = rng.random() < 0.5
        n = _log_int(rng, 1, 64 if tree else 600)
        return {"kind": kind, "requests": n, "rows": _log_int(rng, 2, 100) if tree else 1,
                "prompts": 0 if tree else rng.randint(0, min(n, 9)), "far": _log_int(rng, 10, 8000),
                "page": rng.choice([16, 24, 32, 64]), "tree": tree}
    if kind == "table":
        rot = rng.choice([32, 64, 96, 128, 256])
        return {"kind": kind, "from": rng.choice([0, 0, rng.randint(1, 1000000)]), "rot": rot,
                "positions": _log_int(rng, 64, 131072 * 128 // rot // 2), "factor": rng.choice([1.0, 2.0, 4.0, 8.0, 40.0]),
                "scaling": rng.choice(["none", "linear", "base", "wavelength", "yarn"])}
    if kind == "rotate":
        heads = rng.randrange(len(HEADS))
        rows = rng.randint(1, 8) if rng.random() < 0.3 else _log_int(rng, 9, 2000)
        return {"kind": kind, "heads": heads, "rows": rows, "rot": rng.choice([32, 64, 96, HEADS[heads][2]]),
                "paired": rng.random() < 0.5, "f16": rng.random() < 0.5, "norm": rng.random() < 0.6,
                "padded": rng.choice([0, 0, rows // 5])}
    if kind == "tree":
        tree = rng.random() < 0.6
        sequences = _log_int(rng, 1, 24)
        rows = _log_int(rng, 2, 64) if tree else rng.choice([1, 1, _log_int(rng, 2, 300)])
        far = _log_int(rng, 20, min(60000, 131072 * 60 // (rows * sequences), 16000 * 24 // sequences))
        return {"kind": kind, "heads": rng.randrange(len(HEADS)), "sequences": sequences, "rows": rows,
                "near": rng.choice([0, far // 20, far]), "far": far, "page": rng.choice([0, 16, 24, 64]), "tree": tree}
    if kind == "select":
        beams, used = rng.choice([1, 2, 4, 5, 8, 16]), _log_int(rng, 200, VOCAB)
        return {"kind": kind, "batch": _log_int(rng, 1, max(1, 128 * 75000 // (max(used, 75000) * beams))), "beams": beams,
                "k": min(rng.choice([beams, 2 * beams, 3 * beams, 20]), 64), "used": used, "done": rng.random() < 0.5}
    return {"kind": kind, "layers": rng.choice([8, 20, 40]), "heads": rng.randrange(2), "lists": _log_int(rng, 1, 32),
            "page": rng.choice([16, 24, 64])}


# ---- the cases' lengths and trees, by the case alone --------------------------------------------
def _part(i):
    return math.modf(0.6180339887498949 * (i + 1))[0]


def _lengths(c):
    """(cached keys, rows) of each sequence"""
    if c["kind"] == "tree":
        n = c["sequences"]
        spread = c["far"] - c["near"]
        cached = [c["near"] + int(spread * _part(b)) for b in range(n)] if n > 1 else [c["far"]]
        rows = [c["rows"] if b % 3 == 0 or c["rows"] == 1 else max(1, int(c["rows"] * (0.5 + _part(7 * b) / 2))) for b in range(n)]
        return cached, rows
    cached, rows = [], []
    for b in range(c["requests"]):
        done, prompt = b % 11 == 10, b < c["prompts"]
        cached.append(0 if done or prompt else int(c["far"] * _part(b)))
        rows.append(0 if done else 100 + int(1900 * _part(5 * b)) if prompt else c["rows"] if b % 3 else max(1, c["rows"] // 2))
    return cached, rows


def _parents(b, n):
    """node 0 is the text's next token, every other one the child of one before it"""
    return [-1] + [((i * 2654435761 + b * 40503 >> 7) % i) ** 2 // i for i in range(1, n)]


# ---- inputs -------------------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(g, *shape, mean=0.0, std=1.0, dtype=torch.float32):
    return torch.empty(shape, device="cuda", dtype=dtype).normal_(mean, std, generator=g)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _words(rows):
    return max(1, -(-max(rows) // 32))


def _new_ints(*shape):
    return torch.full(shape, -1, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    c, g = dict(case), _gen(seed)
    s = {"c": c, "stream": torch.cuda.current_stream().cuda_stream}
    {"plan": _prepare_plan, "table": _prepare_table, "rotate": _prepare_rotate, "tree": _prepare_tree,
     "select": _prepare_select, "move": _prepare_move}[c["kind"]](s, c, g)
    return s


def _prepare_plan(s, c, g):
    cached, rows = _lengths(c)
    n, page = c["requests"], c["page"]
    # the pages that a request holds from the steps before; one that is done still holds some
    held = [-(-k // page) + (3 if r == 0 else b % 2) for b, (k, r) in enumerate(zip(cached, rows))]
    most = max(max(-(-(k + r) // page) for k, r in zip(cached, rows)), max(held))
    free = sum(-(-(k + r) // page) for k, r in zip(cached, rows)) + 40
    total = sum(held) + free
    order = torch.randperm(total, generator=g, device="cuda", dtype=torch.int32)
    tables, at = [], 0
    for h in held:
        tables.append(torch.cat([order[at:at + h], torch.full((most - h,), -1, dtype=torch.int32, device="cuda")]))
        at += h
    s["tables"] = torch.stack(tables)
    s["ring"] = torch.full((total,), -1, dtype=torch.int32, device="cuda")
    head = total - free // 2  # the ring's free pages run over its end
    s["ring"][(head + torch.arange(free, device="cuda")) % total] = order[at:]
    s["ring_at"], s["cached"], s["added"], s["held"] = _ints([head, free]), _ints(cached), _ints(rows), _ints(held)
    s["rows"], s["words"], s["pages"] = sum(rows), _words(rows), total
    T = s["rows"]
    s["parent"] = _ints([p for b, r in enumerate(rows) if r for p in _parents(b, r)]) if c["tree"] else None
    s["held_out"], s["ring_at_out"], s["row_start"] = _new_ints(n), _new_ints(2), _new_ints(n + 1)
    s["seq"], s["slot"], s["pos"] = _new_ints(T), _new_ints(T), _new_ints(T)
    s["mask"] = _new_ints(T, s["words"]) if c["tree"] else None


def _prepare_table(s, c, g):
    # no inputs but the numbers that say how the frequencies are scaled; another seed, another base
    s["theta"] = float(torch.randint(10000, 1000001, (1,), generator=g, device="cuda"))
    s["table"] = torch.empty(c["positions"], 2, c["rot"] // 2, device="cuda")


def _prepare_rotate(s, c, g):
    qh, kvh, hd = HEADS[c["heads"]]
    T, n = c["rows"], c["rows"] + 100
    s["qkv"] = _normal(g, T, (qh + 2 * kvh) * hd, dtype=torch.float16 if c["f16"] else torch.float32)
    s["q_norm"], s["k_norm"] = (_normal(g, hd, mean=1.0, std=0.02) if c["norm"] else None for _ in range(2))
    positions = 8192
    angle = torch.arange(positions, dtype=torch.float64, device="cuda")[:, None] * 1e6 ** (
        -2.0 * torch.arange(c["rot"] // 2, dtype=torch.float64, device="cuda") / c["rot"])
    s["rope"] = torch.stack([angle.cos(), angle.sin()], 1).float()
    s["pos"] = torch.randint(0, positions, (T,), generator=g, device="cuda", dtype=torch.int32)
    s["slot"] = torch.randperm(n, generator=g, device="cuda", dtype=torch.int32)[:T].contiguous()
    s["slot"][T - c["padded"]:] = -1
    s["k"], s["v"] = (_normal(g, kvh, n, hd, dtype=torch.float16) for _ in range(2))
    s["q"] = torch.empty(T, qh, hd, device="cuda")


def _prepare_tree(s, c, g):
    qh, kvh, hd = HEADS[c["heads"]]
    cached, rows = _lengths(c)
    T, n, page = sum(rows), c["sequences"], c["page"]
    keys = [a + b for a, b in zip(cached, rows)]
    s["lengths"] = cached, rows
    s["q"] = _normal(g, T, qh, hd)
    s["kv_len"] = max(keys)
    if page:
        pages = [-(-k // page) for k in keys]
        s["pages"] = sum(pages) + 5
        order = torch.randperm(s["pages"], generator=g, device="cuda", dtype=torch.int32)
        s["tables"], at = torch.zeros(n, max(pages), dtype=torch.int32, device="cuda"), 0
        for b, k in enumerate(pages):
            s["tables"][b, :k] = order[at:at + k]
            at += k
        cache = s["pages"] * page
    else:  # a stretch of the cache for each sequence
        s["tables"], s["pages"], cache = None, 0, n * max(keys)
    s["k"], s["v"] = (_normal(g, kvh, cache, hd, dtype=torch.float16) for _ in range(2))
    starts = [0]
    for r in rows:
        starts.append(starts[-1] + r)
    s["row_start"], s["cached"] = _ints(starts), _ints(cached)
    s["words"], s["mask"] = _words(rows), None
    if c["tree"]:
        mask = []
        for b, r in enumerate(rows):
            bits = []
            for i, p in enumerate(_parents(b, r)):
                bits.append(1 << i | (bits[p] if p >= 0 else 0))
            mask += [[(x >> 32 * w & 0xFFFFFFFF) - ((x >> 32 * w + 31 & 1) << 32) for w in range(s["words"])] for x in bits]
        s["mask"] = _ints(mask)
    s["out"] = torch.empty(T, qh, hd, device="cuda", dtype=torch.float16)


def _prepare_select(s, c, g):
    rows, used = c["batch"] * c["beams"], c["used"]
    x = _normal(g, rows, used, std=2.0)
    likely = torch.randint(0, used, (rows,), generator=g, device="cuda")
    x.scatter_add_(1, likely[:, None], torch.empty(rows, 1, device="cuda").uniform_(0.0, 12.0, generator=g))
    s["logits"] = x
    s["cum"] = torch.empty(rows, device="cuda").uniform_(-20.0, -10.0, generator=g)
    s["eos"] = used // 2
    s["done"] = (torch.rand(rows, generator=g, device="cuda") < 0.2).to(torch.int32) if c["done"] else None
    s["ids"], s["from"] = _new_ints(c["batch"], c["k"]), _new_ints(c["batch"], c["k"])
    s["scores"] = torch.empty(c["batch"], c["k"], device="cuda")


def _prepare_move(s, c, g):
    _, kvh, hd = HEADS[c["heads"]]
    page, lists = c["page"], c["lists"]
    rows = 2 * lists * page
    s["k"], s["v"] = (_normal(g, c["layers"], kvh, rows, hd, dtype=torch.float16) for _ in range(2))
    # list i: the first rows of one page to another's, the pages read and the pages written apart
    order = torch.randperm(2 * lists, generator=g, device="cuda").tolist()
    origin, to = [], []
    for i in range(lists):
        used = 1 + int((page - 1) * _part(i))
        origin.append([order[i * 3 // 4] * page + r if r < used else -1 for r in range(page)])
        to.append([order[lists + i] * page + r if r < used else -1 for r in range(page)])
    s["origin"], s["to"], s["cache_rows"] = _ints(origin), _ints(to), rows


# ---- the library's entries ----------------------------------------------------------------------
def _p(t):
    return None if t is None else t.data_ptr()


def _bind(s):
    """The call of this state: a program fixes its buffers, sizes and workspace once and then repeats the call."""
    import importlib
    mi = importlib.import_module("intel-arc-inference-server_amd")
    c, st, L = s["c"], s["stream"], mi.lib()
    ref = mi.C.byref

    def workspace(n):
        s["ws"] = torch.empty(max(n, 1), device="cuda", dtype=torch.uint8)
        return _p(s["ws"]), n

    def shape(rot):
        qh, kvh, hd = HEADS[c["heads"]]
        return mi.AttnShape(qh, kvh, hd, rot, 0, (qh + 2 * kvh) * hd, qh * hd, (qh + kvh) * hd, hd ** -0.5, EPS, 0)

    if c["kind"] == "plan":
        s["struct"] = mi.BlockPlan(
            requests=c["requests"], rows=s["rows"], page=c["page"], n_pages=s["pages"], table_stride=s["tables"].shape[1],
            ring_len=len(s["ring"]), words=s["words"] if c["tree"] else 0, cached=_p(s["cached"]), added=_p(s["added"]),
            held=_p(s["held"]), held_out=_p(s["held_out"]), tables=_p(s["tables"]), ring=_p(s["ring"]),
            ring_at=_p(s["ring_at"]), ring_at_out=_p(s["ring_at_out"]), parent=_p(s["parent"]), row_start=_p(s["row_start"]),
            seq=_p(s["seq"]), slot=_p(s["slot"]), pos=_p(s["pos"]), mask=_p(s["mask"]), flag=None)
        args = ("mi_block_tables", ref(s["struct"]), *workspace(L.mi_block_tables_ws(c["requests"])), st)
        outs = _plan_outputs(*(s[k] for k in ("tables", "ring", "held_out", "ring_at_out", "row_start", "seq", "slot", "pos", "mask")))
    elif c["kind"] == "table":
        s["struct"] = mi.Rope(rot_dim=c["rot"], theta=s["theta"], scaling=getattr(mi, "ROPE_" + c["scaling"].upper()),
                              factor=c["factor"], original=4096, low=1.0, high=32.0 if c["scaling"] == "yarn" else 4.0,
                              attention=0.0, divisors=None)
        args = ("mi_rope_table", ref(s["struct"]), c["from"], c["positions"], _p(s["table"]), st)
        outs = s["table"]
    elif c["kind"] == "rotate":
        sh = s["struct"] = shape(c["rot"])
        n, hd = s["k"].shape[1:]
        args = ("mi_rope_rows", _p(s["qkv"]), mi.OUT_F16 if c["f16"] else mi.OUT_F32, sh.qkv_n, c["rows"], _p(s["pos"]), 0,
                _p(s["slot"]), n, ref(sh), int(c["paired"]), _p(s["q_norm"]), _p(s["k_norm"]), _p(s["rope"]), len(s["rope"]),
                _p(s["q"]), _p(s["k"]), _p(s["v"]), hd, n * hd, None, st)
        outs = s["q"], s["k"], s["v"]
    elif c["kind"] == "tree":
        sh = shape(HEADS[c["heads"]][2])
        n, hd, T = *s["k"].shape[1:], len(s["q"])
        batch = mi.AttnBatch(
            sequences=c["sequences"], kv_len=s["kv_len"], row_start=_p(s["row_start"]), cached=_p(s["cached"]),
            tables=_p(s["tables"]), table_stride=s["kv_len"] if s["tables"] is None else s["tables"].shape[1], page=c["page"],
            n_pages=s["pages"], mask=_p(s["mask"]), words=s["words"] if c["tree"] else 0)
        s["struct"] = sh, batch
        args = ("mi_attn_tree", _p(s["q"]), _p(s["k"]), _p(s["v"]), hd, n * hd, T, ref(sh), ref(batch),
                *workspace(L.mi_attn_tree_ws(T, c["sequences"], ref(sh))), _p(s["out"]), None, st)
        outs = s["out"]
    elif c["kind"] == "select":
        sizes = c["batch"], c["beams"], c["used"], c["k"]
        args = ("mi_beam_select", _p(s["logits"]), c["used"], _p(s["cum"]), _p(s["done"]), s["eos"], *sizes, _p(s["ids"]),
                _p(s["from"]), _p(s["scores"]), *workspace(L.mi_beam_select_ws(*sizes)), st)
        outs = s["ids"], s["from"], s["scores"]
    else:
        layers, kvh, n, hd = s["k"].shape
        args = ("mi_kv_move", _p(s["k"]), _p(s["v"]), layers, kvh * n * hd, hd, n * hd, kvh, hd, n, _p(s["origin"]), _p(s["to"]),
                c["lists"], c["page"], None, st)
        outs = s["k"], s["v"]
    return mi.call, args, outs


# ---- one pass -----------------------------------------------------------------------------------
def _plan_outputs(tables, ring, held, ring_at, row_start, seq, slot, pos, mask):
    return {"tables": tables, "ring": ring, "held": held, "ring_at": ring_at, "row_start": row_start, "seq": seq, "slot": slot,
            "pos": pos, "mask": mask if mask is not None else torch.zeros(0, dtype=torch.int32)}


def run(s):
    if own:
        if "call" not in s:
            s["call"] = _bind(s)
        call, args, outs = s["call"]
        call(*args)
        return outs
    return {"plan": _plain_plan, "table": _plain_table, "rotate": _plain_rotate, "tree": _plain_tree, "select": _plain_select,
            "move": _plain_move}[s["c"]["kind"]](s)


def _plain_plan(s):
    c, T = s["c"], s["rows"]
    page, size = c["page"], len(s["ring"])
    cached, added, held = (s[k].long() for k in ("cached", "added", "held"))
    need = (cached + added + page - 1) // page
    taken, back = (need - held).clamp(min=0), (held - need).clamp(min=0)
    first_taken, first_back = taken.cumsum(0) - taken, back.cumsum(0) - back
    head, count = s["ring_at"].long()
    ring, tables = s["ring"], s["tables"]
    i = torch.arange(tables.shape[1], device="cuda")[None, :]
    at = (head + first_taken[:, None] + (i - held[:, None])) % size
    tables = torch.where((i >= held[:, None]) & (i < need[:, None]), ring[at], tables)
    gives = (i >= need[:, None]) & (i < held[:, None])
    at = (head + count + first_back[:, None] + (i - need[:, None])) % size
    room = torch.cat([ring, ring.new_zeros(1)])  # (one place behind the ring for what is not given back)
    ring = room.scatter(0, torch.where(gives, at, torch.full_like(at, size)).flatten(), tables.flatten())[:size]
    row_start = torch.cat([added.new_zeros(1), added.cumsum(0)])
    t = torch.arange(T, device="cuda")
    seq = torch.searchsorted(row_start, t, right=True) - 1
    inside = t - row_start[seq]
    key = cached[seq] + inside
    slot = tables[seq, key // page].long() * page + key % page
    mask = None
    if s["parent"] is not None:
        # ancestors by doubling: who is 2^n steps above, and which nodes lie on the way
        above = torch.where(s["parent"] >= 0, s["parent"].long() + row_start[seq], torch.full_like(t, T))
        above = torch.cat([above, above.new_full((1,), T)])
        bits = torch.zeros(T + 1, 32 * s["words"], dtype=torch.bool, device="cuda")
        bits[t, inside] = True
        for _ in range(max(1, (32 * s["words"] - 1).bit_length())):
            bits = bits | bits[above]
            above = above[above]
        bits = bits[:T]
        key = cached[seq] + bits.sum(1) - 1
        power = torch.ones(32, dtype=torch.int64, device="cuda") << torch.arange(32, device="cuda")
        mask = (bits.view(T, s["words"], 32) * power).sum(2).to(torch.int32)
    new_at = torch.stack([(head + taken.sum()) % size, count - taken.sum() + back.sum()])
    return _plan_outputs(tables, ring, *(x.to(torch.int32) for x in (need, new_at, row_start, seq, slot, key)), mask)


def _frequencies(c, theta):
    """f_i in 64 bits, and what the cosines and sines are multiplied with"""
    r, by = c["rot"], c["factor"]
    i = torch.arange(r // 2, dtype=torch.float64, device="cuda")
    if c["scaling"] == "base":
        theta = theta * by ** (r / (r - 2))
    f = theta ** (-2.0 * i / r)
    if c["scaling"] == "linear":
        return f / by, 1.0
    if c["scaling"] == "wavelength":
        # turns within the 4096 positions of training: below 1 stretched, from 4 on as they are, between them mixed
        turns = 4096.0 * f / (2.0 * math.pi)
        part = ((turns - 1.0) / 3.0).clamp(0.0, 1.0)
        return (1.0 - part) * f / by + part * f, 1.0
    if c["scaling"] == "yarn":
        lo, hi = (r * math.log(4096.0 / (turns * 2.0 * math.pi)) / (2.0 * math.log(theta)) for turns in (32.0, 1.0))
        lo, hi = max(math.floor(lo), 0), min(math.ceil(hi), r - 1)
        part = ((i - lo) / max(hi - lo, 0.001)).clamp(0.0, 1.0)
        return part * f / by + (1.0 - part) * f, 0.1 * math.log(by) + 1.0 if by > 1.0 else 1.0
    return f, 1.0


def _plain_table(s):
    c = s["c"]
    f, much = _frequencies(c, s["theta"])
    p = torch.arange(c["from"], c["from"] + c["positions"], dtype=torch.float64, device="cuda")
    angle = p[:, None] * f
    return torch.stack([(angle.cos() * much).float(), (angle.sin() * much).float()], 1)


def _pairs(c, hd):
    i = torch.arange(c["rot"] // 2, device="cuda")
    return (2 * i, 2 * i + 1) if c["paired"] else (i, i + c["rot"] // 2)


def _plain_rotate(s):
    c = s["c"]
    qh, kvh, hd = HEADS[c["heads"]]
    T = c["rows"]
    q, k, v = s["qkv"].float().view(T, qh + 2 * kvh, hd).split([qh, kvh, kvh], 1)
    if c["norm"]:
        q = q / torch.sqrt((q * q).mean(2, keepdim=True) + EPS) * s["q_norm"]
        k = k / torch.sqrt((k * k).mean(2, keepdim=True) + EPS) * s["k_norm"]
    a, b = _pairs(c, hd)
    cos, sin = s["rope"][s["pos"].long()][:, None].unbind(2)
    out = []
    for x in (q, k):
        y = x.clone()
        y[:, :, a] = x[:, :, a] * cos - x[:, :, b] * sin
        y[:, :, b] = x[:, :, b] * cos + x[:, :, a] * sin
        out.append(y)
    live = T - c["padded"]
    at = s["slot"][:live].long()
    ck, cv = s["k"].clone(), s["v"].clone()
    ck[:, at] = out[1][:live].transpose(0, 1).half()
    cv[:, at] = v[:live].transpose(0, 1).half()
    return out[0], ck, cv


def _seen(s, b):
    """[rows, keys] of sequence b"""
    cached, rows = (x[b] for x in s["lengths"])
    i = torch.arange(rows, device="cuda")
    if s["mask"] is None:
        tree = i[None, :] <= i[:, None]
    else:
        first = sum(s["lengths"][1][:b])
        tree = (s["mask"][first:first + rows][:, i // 32] >> (i % 32).to(torch.int32) & 1).bool()
    return torch.cat([torch.ones(rows, cached, dtype=torch.bool, device="cuda"), tree], 1)


def _rows_of_cache(s, b):
    j = torch.arange(sum(x[b] for x in s["lengths"]), device="cuda")
    if s["tables"] is None:
        return b * s["kv_len"] + j
    return s["tables"][b].long()[j // s["c"]["page"]] * s["c"]["page"] + j % s["c"]["page"]


def _plain_tree(s):
    qh, kvh, hd = HEADS[s["c"]["heads"]]
    first, parts = 0, []
    for b, rows in enumerate(s["lengths"][1]):
        at, seen = _rows_of_cache(s, b), _seen(s, b)
        k, v = s["k"][:, at].float(), s["v"][:, at].float()
        q = s["q"][first:first + rows].view(rows, kvh, qh // kvh, hd).permute(1, 2, 0, 3).reshape(kvh, qh // kvh * rows, hd)
        w = ((q @ k.transpose(1, 2).contiguous()) * hd ** -0.5).view(qh, rows, len(at))
        w = torch.where(seen, w, torch.full_like(w, -math.inf))
        e = torch.exp(w - w.amax(2, keepdim=True))
        o = (e.view(kvh, qh // kvh * rows, len(at)) @ v).view(qh, rows, hd) / e.sum(2, keepdim=True)
        parts.append(o.permute(1, 0, 2).half())
        first += rows
    return torch.cat(parts)


def _plain_select(s):
    c = s["c"]
    W, used, n = c["beams"], c["used"], min(c["k"], c["used"])
    x = s["logits"] + 0.0  # (-0 counts as 0)
    # an integer key for each token in its row's order: the larger logit, then the lower index
    bits = x.view(torch.int32)
    key = ((bits ^ ((bits >> 31) & 0x7FFFFFFF)).long() << 32) + (0xFFFFFFFF - torch.arange(used, device="cuda"))
    ids = 0xFFFFFFFF - (key.topk(n, 1).values & 0xFFFFFFFF)
    wide = x.double()
    most = wide.amax(1, keepdim=True)
    score = wide.gather(1, ids) - most - (wide - most).exp().sum(1, keepdim=True).log() + s["cum"].double()[:, None]
    if s["done"] is not None:  # a beam at its end goes on as it is
        only = torch.full_like(score, -math.inf)
        only[:, 0] = s["cum"].double()
        score = torch.where(s["done"][:, None] != 0, only, score)
        ids = torch.where(s["done"][:, None] != 0, torch.full_like(ids, s["eos"]), ids)
    score, ids = score.view(c["batch"], W * n), ids.view(c["batch"], W * n)
    score, place = score.sort(dim=1, descending=True, stable=True)
    k = min(c["k"], W * n)
    score, place = score[:, :k], place[:, :k]
    out = [torch.full((c["batch"], c["k"]), fill, dtype=dt, device="cuda")
           for fill, dt in ((-1, torch.int32), (-1, torch.int32), (-math.inf, torch.float32))]
    for o, v in zip(out, (ids.gather(1, place), place // n, score)):
        o[:, :k] = torch.where(score > -math.inf, v.to(o.dtype), o[:, :k])
    return tuple(out)


def _plain_move(s):
    live = s["to"].flatten() >= 0
    # (what no row goes to is a place behind the cache)
    rows = s["cache_rows"]
    at = torch.where(live, s["to"].flatten().long(), torch.full_like(live, rows, dtype=torch.int64))
    whence = s["origin"].flatten().long().clamp(min=0)
    out = []
    for x in (s["k"], s["v"]):
        room = torch.cat([x, x[:, :, :1]], 2)
        room[:, :, at] = x[:, :, whence]
        out.append(room[:, :, :rows].contiguous())
    return tuple(out)


# ---- what a pass cannot do without --------------------------------------------------------------
def work(case):
    c = case
    if c["kind"] == "plan":
        cached, rows = _lengths(c)
        T, page = sum(rows), c["page"]
        words = _words(rows) + 1 if c["tree"] else 0  # (the masks and the parents)
        new = sum(-(-(k + r) // page) - -(-k // page) for k, r in zip(cached, rows))
        return {"bytes": 4 * (5 * c["requests"] + T * (3 + words) + 2 * new), "flops": 0}
    if c["kind"] == "table":
        n = c["positions"] * c["rot"] // 2
        return {"bytes": 8 * n, "flops": 30 * n}
    if c["kind"] == "rotate":
        qh, kvh, hd = HEADS[c["heads"]]
        live = c["rows"] - c["padded"]
        return {"bytes": c["rows"] * (qh * hd * (6 if c["f16"] else 8) + 4 * c["rot"] + 8) +
                live * 2 * kvh * hd * (4 if c["f16"] else 6), "flops": c["rows"] * (qh + kvh) * (4 * hd + 3 * c["rot"])}
    if c["kind"] == "tree":
        qh, kvh, hd = HEADS[c["heads"]]
        cached, rows = _lengths(c)
        pairs = 0
        for b, (k, r) in enumerate(zip(cached, rows)):
            depth = []
            for i, p in enumerate(_parents(b, r) if c["tree"] else range(-1, r - 1)):
                depth.append(1 + (depth[p] if p >= 0 else 0))
            pairs += k * r + sum(depth)
        return {"bytes": 6 * sum(rows) * qh * hd + 4 * (sum(cached) + sum(rows)) * kvh * hd, "flops": 4 * pairs * qh * hd}
    if c["kind"] == "select":
        n = c["batch"] * c["beams"] * c["used"]
        return {"bytes": 4 * n + 12 * c["batch"] * c["k"], "flops": 4 * n}
    _, kvh, hd = HEADS[c["heads"]]
    moved = sum(1 + int((c["page"] - 1) * _part(i)) for i in range(c["lists"]))
    return {"bytes": 8 * c["layers"] * kvh * hd * moved, "flops": 0}


# ---- the definitions in 64 bits -----------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return {"plan": _exact_plan, "table": _exact_table, "rotate": _exact_rotate, "tree": _exact_tree, "select": _exact_select,
            "move": _exact_move}[case["kind"]](s)


def _exact_plan(s):
    """request by request and row by row"""
    c = s["c"]
    page = c["page"]
    cached, added, held, ring, tables = (s[k].tolist() for k in ("cached", "added", "held", "ring", "tables"))
    head, count = s["ring_at"].tolist()
    parent = s["parent"].tolist() if s["parent"] is not None else None
    back, row_start, seq, slot, pos, mask, new_held = [], [0], [], [], [], [], []
    size, taken = len(ring), 0
    for b in range(c["requests"]):
        have = held[b]
        while have * page < cached[b] + added[b]:
            tables[b][have] = ring[(head + taken) % size]
            have, taken = have + 1, taken + 1
        while (have - 1) * page >= cached[b] + added[b] and have > 0:
            have -= 1
        back += tables[b][have:held[b]]
        new_held.append(have)
        bits = []
        for i in range(added[b]):
            key = cached[b] + i
            seq.append(b)
            slot.append(tables[b][key // page] * page + key % page)
            if parent is None:
                pos.append(key)
                continue
            up = parent[row_start[b] + i]
            bits.append({i} | (bits[up] if up >= 0 else set()))
            pos.append(cached[b] + len(bits[i]) - 1)
            words = [sum(1 << n % 32 for n in bits[i] if n // 32 == w) for w in range(s["words"])]
            mask.append([w - (1 << 32) if w >> 31 else w for w in words])
        row_start.append(row_start[b] + added[b])
    for i, p in enumerate(back):
        ring[(head + count + i) % size] = p
    now = [(head + taken) % size, count - taken + len(back)]
    return _plan_outputs(*(_ints(x) for x in (tables, ring, new_held, now, row_start, seq, slot, pos)),
                         _ints(mask) if parent is not None else None)


def _exact_table(s):
    c = s["c"]
    r, by, theta = c["rot"], c["factor"], s["theta"]
    f, much = [], 1.0
    for i in range(r // 2):
        plain = math.exp(-2.0 * i / r * math.log(theta))
        if c["scaling"] == "linear":
            f.append(plain / by)
        elif c["scaling"] == "base":
            f.append(math.exp(-2.0 * i / r * (math.log(theta) + math.log(by) * r / (r - 2))))
        elif c["scaling"] == "wavelength":
            length = 2.0 * math.pi / plain
            if length > 4096.0:
                f.append(plain / by)
            elif length < 4096.0 / 4.0:
                f.append(plain)
            else:
                mix = (4096.0 / length - 1.0) / (4.0 - 1.0)
                f.append((1.0 - mix) * plain / by + mix * plain)
        elif c["scaling"] == "yarn":
            # the (fractional) pair that turns n times over the positions of training
            def pair(n):
                return r / 2.0 * math.log(4096.0 / (2.0 * math.pi * n)) / math.log(theta)
            lo, hi = max(math.floor(pair(32.0)), 0), min(math.ceil(pair(1.0)), r - 1)
            ramp = min(max((i - lo) / (hi - lo if hi > lo else 0.001), 0.0), 1.0)
            f.append(plain * (1.0 - ramp) + plain / by * ramp)
            much = 1.0 + 0.1 * math.log(max(by, 1.0))
        else:
            f.append(plain)
    p = torch.arange(c["positions"], dtype=torch.float64, device="cuda") + c["from"]
    angle = torch.outer(p, torch.tensor(f, dtype=torch.float64, device="cuda"))
    return torch.stack([torch.cos(angle), torch.sin(angle)], dim=1) * much


def _exact_rotate(s):
    c = s["c"]
    qh, kvh, hd = HEADS[c["heads"]]
    T, r = c["rows"], c["rot"]
    x = s["qkv"].double().view(T, qh + 2 * kvh, hd)
    rows = s["rope"].double()[s["pos"].long()]
    turn = torch.complex(rows[:, 0], rows[:, 1])[:, None]  # a pair as a complex number, turned

    def turned(x, weight):
        if weight is not None:
            x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * weight.double()
        part = x[..., :r]
        if c["paired"]:
            z = torch.view_as_complex(part.reshape(T, -1, r // 2, 2).contiguous()) * turn
            part = torch.view_as_real(z).flatten(-2)
        else:
            z = torch.complex(part[..., :r // 2].contiguous(), part[..., r // 2:].contiguous()) * turn
            part = torch.cat([z.real, z.imag], -1)
        return torch.cat([part, x[..., r:]], -1)

    k, v = s["k"].double(), s["v"].double()
    new_k, new_v = turned(x[:, qh:qh + kvh], s["k_norm"]), x[:, qh + kvh:]
    for t, row in enumerate(s["slot"].tolist()):
        if row >= 0:
            k[:, row], v[:, row] = new_k[t], new_v[t]
    return turned(x[:, :qh], s["q_norm"]), k, v


def _exact_tree(s):
    qh, kvh, hd = HEADS[s["c"]["heads"]]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    first = 0
    for b, rows in enumerate(s["lengths"][1]):
        at, hidden = _rows_of_cache(s, b), ~_seen(s, b)
        for h in range(qh):
            k, v = s["k"][h * kvh // qh][at].double(), s["v"][h * kvh // qh][at].double()
            w = torch.mm(s["q"][first:first + rows, h].double(), k.t().contiguous()) / math.sqrt(hd)
            w[hidden] = -math.inf
            out[first:first + rows, h] = torch.mm(torch.softmax(w, dim=1), v)
        first += rows
    return out


def _exact_select(s):
    c = s["c"]
    ids, beams, scores = [], [], []
    for b in range(c["batch"]):
        at = slice(b * c["beams"], (b + 1) * c["beams"])
        lp = torch.log_softmax(s["logits"][at].double(), dim=1) + s["cum"][at].double()[:, None]
        if s["done"] is not None:
            for w in s["done"][at].nonzero().flatten().tolist():
                lp[w] = -math.inf
                lp[w, s["eos"]] = s["cum"][at][w].double()
        best = torch.sort(lp.flatten(), descending=True, stable=True)
        n = min(c["k"], best.values.numel())
        none = torch.isinf(best.values[:n])
        fill = torch.full((c["k"] - n,), -1, dtype=torch.int64, device="cuda")
        ids.append(torch.cat([(best.indices[:n] % c["used"]).masked_fill(none, -1), fill]))
        beams.append(torch.cat([(best.indices[:n] // c["used"]).masked_fill(none, -1), fill]))
        scores.append(torch.cat([best.values[:n], torch.full((c["k"] - n,), -math.inf, dtype=torch.float64, device="cuda")]))
    return torch.stack(ids).to(torch.int32), torch.stack(beams).to(torch.int32), torch.stack(scores)


def _exact_move(s):
    """list by list"""
    out = []
    for x in (s["k"], s["v"]):
        y = x.double()
        for origin, to in zip(s["origin"].tolist(), s["to"].tolist()):
            n = sum(r >= 0 for r in to)  # (the rows that go stand at the front)
            y[:, :, to[:n]] = x[:, :, origin[:n]].double()
        out.append(y)
    return tuple(out)
