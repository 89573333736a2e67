"""Differential attention and the pages of a key-value cache, as they are measured.

A case is a dict of plain values with a "path":

* "train":   forward and backward of differential attention on a dense batch
* "varlen":  the same on a packed batch of sequences of mixed lengths
* "prompt":  forward only, no gradients
* "cache":   differential attention with a key-value cache: decode steps and prompt chunks, with an append
* "fork":    rows of a paged cache end, others fork from their parents and all get room for the next tokens
* "compact": the pages in use move to the front of the pool

Differential attention of one head: q and k hold two maps in the two halves of their channels,
o = (softmax(scale q1 k1^T) - lam softmax(scale q2 k2^T)) v with scale = (dim / 2) ** -0.5.

Inputs are normal with unit variance, as projections after a normalisation are; lam is near the 0.2 to 0.8 that
trained layers start from.  Lengths of mixed batches and the tables of a cache follow from the case alone (its
"lengths" number), values from the seed.
"""

import math
import os
import random
import sys

import torch

own = False

PAGE = 256  # tokens of a cache page
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
DEVICE = "cuda"


def _interface():
    folder = os.path.join(os.getcwd(), "flash-attention-turing_amd")
    if folder not in sys.path:
        sys.path.insert(0, folder)
    import flash_attention_interface

    return flash_attention_interface


# ---------------------------------------------------------------------------
# Cases.


def _dense(name, path, batch, seqlen_q, seqlen_k, heads, heads_k, dim, causal, lam, dtype):
    return {"name": name, "path": path, "batch": batch, "seqlen_q": seqlen_q, "seqlen_k": seqlen_k, "heads": heads,
            "heads_k": heads_k, "dim": dim, "causal": causal, "lam": lam, "dtype": dtype}


def _varlen(name, batch, shortest, longest, heads, heads_k, dim, causal, lam, dtype, lengths):
    return {"name": name, "path": "varlen", "batch": batch, "shortest": shortest, "longest": longest, "heads": heads,
            "heads_k": heads_k, "dim": dim, "causal": causal, "lam": lam, "dtype": dtype, "lengths": lengths}


def _cache(name, batch, queries, heads, heads_k, dim, shortest, longest, layout, lam, dtype, lengths):
    """queries: query tokens a sequence, as many are appended.  shortest, longest: tokens in the cache before."""
    return {"name": name, "path": "cache", "batch": batch, "queries": queries, "heads": heads, "heads_k": heads_k,
            "dim": dim, "shortest": shortest, "longest": longest, "layout": layout, "lam": lam, "dtype": dtype,
            "lengths": lengths}


def _fork(name, parents, children, heads_k, dim, shortest, longest, dtype, lengths):
    """children: rows that fork from each parent."""
    return {"name": name, "path": "fork", "parents": parents, "children": children, "heads_k": heads_k, "dim": dim,
            "shortest": shortest, "longest": longest, "dtype": dtype, "lengths": lengths}


def _compact(name, pages, rows, per_row, shared, heads_k, dim, dtype, lengths):
    """rows of per_row pages each, the first `shared` of them common to all rows, anywhere in a pool of `pages`."""
    return {"name": name, "path": "compact", "pages": pages, "rows": rows, "per_row": per_row, "shared": shared,
            "heads_k": heads_k, "dim": dim, "dtype": dtype, "lengths": lengths}


def listed():
    return [
        # The shortest useful training call: one short text, where launches are what a step costs.
        _dense("train_one", "train", 1, 77, 77, 8, 8, 64, True, "head", "fp16"),
        # The benchmark's headline batch as a differential layer, one lam for the layer.
        _dense("train_4k", "train", 4, 4096, 4096, 16, 16, 128, True, "layer", "bf16"),
        # One long text on each GPU, grouped heads, a lam for each token and head.
        _dense("train_long", "train", 1, 8192, 8192, 32, 8, 128, True, "token", "fp16"),
        # A packed batch of documents of mixed lengths, grouped heads of 64 channels.
        _varlen("train_varlen", 16, 100, 2048, 16, 4, 64, True, "head", "bf16", 2),
        # A short prompt's only pass: scoring, or the first answer of a chat.
        _dense("prompt_short", "prompt", 1, 509, 509, 32, 8, 128, True, "layer", "fp16"),
        # One user's next token in a chat.
        _cache("decode_one", 1, 1, 32, 8, 128, 1500, 1500, "contiguous", "layer", "fp16", 3),
        # A serving step: 64 sequences of 1k to 16k tokens in a paged cache.
        _cache("decode_batch", 64, 1, 32, 8, 128, 1024, 16384, "paged", "head", "bf16", 3),
        # The next piece of two long prompts in a paged serving cache (chunked prefill).
        _cache("chunk_paged", 2, 512, 32, 8, 128, 4096, 12000, "paged", "layer", "bf16", 3),
        # A beam search's next step: four beams fork from one of the last step's.
        _fork("fork_beams", 1, 4, 8, 128, 1500, 1500, "fp16", 3),
        # Parallel sampling: 16 prompts of 1k to 8k tokens, 16 answers each.
        _fork("fork_samples", 16, 16, 8, 128, 1000, 8000, "bf16", 3),
        # A small pool between two requests.
        _compact("compact_small", 64, 9, 4, 1, 4, 64, "fp16", 3),
        # A serving pool after many requests of mixed lengths have ended: 1600 pages, half in use.
        _compact("compact_pool", 1600, 96, 9, 1, 8, 128, "bf16", 3),
    ]


HEADS = [(8, 8), (16, 16), (12, 4), (16, 4), (32, 8), (32, 4), (6, 2)]
MOST_FLOPS = 14 * 128 * 16 * 4 * (4096 * 4097 // 2)  # the headline training step
MOST_TOKENS = 64 * 5600  # cache tokens of the serving step


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    path = rng.choice(["train", "train", "varlen", "prompt", "cache", "cache", "cache", "fork", "compact"])
    heads, heads_k = rng.choice(HEADS)
    dim, dtype = rng.choice([64, 128]), rng.choice(["fp16", "bf16"])
    lam, causal = rng.choice(["layer", "head", "token"]), rng.random() < 0.7
    lengths = rng.randrange(1, 1 << 20)
    while True:
        if path in ("train", "prompt"):
            least = 2 if path == "train" else 1  # one key: the gradients of q and k are 0, and rounding all that is there
            q = _spread(rng, least, 6000)
            k = q if rng.random() < 0.6 else _spread(rng, least, 6000)
            case = _dense("", path, _spread(rng, 1, 12), q, k, heads, heads_k, dim, causal, lam, dtype)
        elif path == "varlen":
            longest = _spread(rng, 16, 3000)
            case = _varlen("", _spread(rng, 1, 24), _spread(rng, 1, longest), longest, heads, heads_k, dim, causal, lam,
                           dtype, lengths)
        elif path == "cache":
            queries = 1 if rng.random() < 0.5 else _spread(rng, 1, 700)
            longest = _spread(rng, 16, 40000)
            case = _cache("", _spread(rng, 1, 64), queries, heads, heads_k, dim, _spread(rng, 1, longest), longest,
                          rng.choice(["paged", "paged", "contiguous", "remapped"]), lam, dtype, lengths)
        elif path == "fork":
            longest = _spread(rng, 10, 8000)
            case = _fork("", _spread(rng, 1, 16), _spread(rng, 1, 16), rng.choice([2, 4, 8]), dim,
                         _spread(rng, 1, longest), longest, dtype, lengths)
        else:
            rows, per_row = _spread(rng, 1, 96), _spread(rng, 2, 16)
            shared = rng.randrange(0, per_row)
            used = shared + rows * (per_row - shared)
            pages = int(used * rng.uniform(1.05, 4.0)) + 1
            case = _compact("", pages, rows, per_row, shared, rng.choice([2, 4, 8]), dim, dtype, lengths)
        del case["name"]
        w = work(case)
        if case["path"] == "cache":
            tokens = sum(n + case["queries"] for n in _lengths(case))
            pairs = case["batch"] * case["heads"] * case["queries"] * (case["longest"] + case["queries"])
            ok = tokens * heads_k * dim <= MOST_TOKENS * 8 * 128 and pairs <= 1 << 30
        elif case["path"] == "compact":
            ok = case["pages"] * case["heads_k"] * dim <= 1600 * 8 * 128
        elif case["path"] == "varlen":
            ok = w["flops"] <= MOST_FLOPS and case["batch"] * case["heads"] * case["longest"] ** 2 <= 1 << 30
        else:
            ok = w["flops"] <= MOST_FLOPS
        if ok:
            return case


def _lengths(case):
    """Lengths of a mixed batch, spread over their logarithm; the longest is among them."""
    r = random.Random(case["lengths"])
    low, high = min(case["shortest"], case["longest"]), case["longest"]
    n = case["parents"] if case["path"] == "fork" else case["batch"]
    got = [_spread(r, low, high) for _ in range(n)]
    got[r.randrange(n)] = high
    return got


def _pairs(q, k, causal):
    """Visible (query, key) pairs of one head; causal is aligned at the ends."""
    if not causal:
        return q * k
    first = k - q + 1  # keys that the first query sees
    empty = min(q, max(0, 1 - first))
    return _sum_range(max(first, 1), first + q - 1) if q > empty else 0


def _sum_range(a, b):
    return (a + b) * (b - a + 1) // 2 if b >= a else 0


def work(case):
    path = case["path"]
    dim = case["dim"]
    if path == "fork":
        row = case["heads_k"] * dim * 2
        parents = _lengths(case)
        moved = sum(n % PAGE for n in parents) * case["children"]
        tables = sum(-(-(n + 1) // PAGE) for n in parents) * case["children"]
        return {"bytes": 2 * 2 * moved * row + 4 * 4 * tables, "flops": 0}
    if path == "compact":
        used = case["shared"] + case["rows"] * (case["per_row"] - case["shared"])
        moved = used * (case["pages"] - used) / case["pages"]  # expected, with the pages anywhere
        page = PAGE * case["heads_k"] * dim * 2
        return {"bytes": 2 * 2 * moved * page + 8 * (case["pages"] + case["rows"] * (case["per_row"] + 2)), "flops": 0}
    h, hk = case["heads"], case["heads_k"]
    if path == "cache":
        lengths, n = _lengths(case), case["queries"]
        tokens = sum(lengths) + 2 * case["batch"] * n
        pairs = sum(_pairs(n, x + n, True) for x in lengths)
        return {"bytes": 2 * 2 * tokens * hk * dim + 2 * 2 * case["batch"] * n * h * dim, "flops": 4 * dim * h * pairs}
    if path == "varlen":
        lengths = _lengths(case)
        pairs = sum(_pairs(x, x, case["causal"]) for x in lengths)
        tq = tk = sum(lengths)
    else:
        pairs = case["batch"] * _pairs(case["seqlen_q"], case["seqlen_k"], case["causal"])
        tq, tk = case["batch"] * case["seqlen_q"], case["batch"] * case["seqlen_k"]
    if path == "prompt":
        return {"bytes": 2 * dim * (2 * tq * h + 2 * tk * hk), "flops": 4 * dim * h * pairs}
    return {"bytes": 2 * dim * (4 * tq * h + 4 * tk * hk), "flops": 14 * dim * h * pairs}


# ---------------------------------------------------------------------------
# Inputs.


def _lam(kind, tokens, heads, gen):
    """tokens: the leading sizes of a lam for each token."""
    if kind == "layer":
        return torch.empty((), device=DEVICE).uniform_(0.2, 0.8, generator=gen)
    if kind == "head":
        return torch.empty((heads,), device=DEVICE).uniform_(0.2, 0.8, generator=gen)
    return torch.sigmoid(torch.randn(*tokens, heads, device=DEVICE, generator=gen))


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed)
    dtype, path = DTYPES[case["dtype"]], case["path"]

    def normal(*shape):
        return torch.randn(*shape, device=DEVICE, dtype=dtype, generator=gen)

    if path == "fork":
        return _prepare_fork(case, normal)
    if path == "compact":
        return _prepare_compact(case, normal)
    h, hk, dim = case["heads"], case["heads_k"], case["dim"]
    s = {"path": path, "scale": (dim // 2) ** -0.5}
    if path == "cache":
        b, n, lengths = case["batch"], case["queries"], _lengths(case)
        capacity = -(-(max(lengths) + n) // PAGE) * PAGE
        s["q"], s["k"], s["v"] = normal(b, n, h, dim), normal(b, n, hk, dim), normal(b, n, hk, dim)
        s["lam"] = _lam(case["lam"], (b, n), h, gen)
        s["lens"] = torch.tensor(lengths, dtype=torch.int32, device=DEVICE)
        s["table"] = s["index"] = None
        r = random.Random(case["lengths"] + 1)
        if case["layout"] == "paged":
            need = [-(-(x + n) // PAGE) for x in lengths]
            pages = list(range(sum(need) + 3))
            r.shuffle(pages)
            table = torch.full((b, capacity // PAGE), -1, dtype=torch.int32)
            for i, m in enumerate(need):
                table[i, :m] = torch.tensor([pages.pop() for _ in range(m)], dtype=torch.int32)
            s["table"] = table.to(DEVICE)
            shape = (sum(need) + 3, PAGE, hk, dim)
        elif case["layout"] == "remapped":
            rows = list(range(b + 2))
            r.shuffle(rows)
            s["index"] = torch.tensor(rows[:b], dtype=torch.int32, device=DEVICE)
            shape = (b + 2, capacity, hk, dim)
        else:
            shape = (b, capacity, hk, dim)
        s["k_cache"], s["v_cache"] = normal(*shape), normal(*shape)
        return s
    if path == "varlen":
        lengths = _lengths(case)
        total = (sum(lengths),)
        total_k = total
        cu = [0]
        for x in lengths:
            cu.append(cu[-1] + x)
        s["cu"] = torch.tensor(cu, dtype=torch.int32, device=DEVICE)
        s["longest"] = max(lengths)
    else:
        total, total_k = (case["batch"], case["seqlen_q"]), (case["batch"], case["seqlen_k"])
    s["causal"] = case["causal"]
    s["q"], s["k"], s["v"] = normal(*total, h, dim), normal(*total_k, hk, dim), normal(*total_k, hk, dim)
    s["lam"] = _lam(case["lam"], total, h, gen)
    if path != "prompt":
        s["dout"] = normal(*total, h, dim)
        for name in ("q", "k", "v", "lam"):
            s[name].requires_grad_()
    return s


def _prepare_fork(case, normal):
    """Rows 0 .. parents - 1 are the prompts; the rows after them hold the answers of the last requests, which end."""
    r = random.Random(case["lengths"] + 1)
    lengths, kids = _lengths(case), case["children"]
    rows = case["parents"] * (1 + kids)
    width = max(lengths) // PAGE + 2
    need = [-(-x // PAGE) for x in lengths]
    pages = list(range(sum(need) + rows * 2 + 5))
    refs, table = [0] * len(pages), torch.full((rows, width), -1, dtype=torch.int32)
    r.shuffle(pages)
    lens = [0] * rows
    for i, m in enumerate(need):
        for j in range(m):
            table[i, j] = pages.pop()
            refs[int(table[i, j])] = 1
        lens[i] = lengths[i]
    for i in range(case["parents"], rows):  # an answer of up to a page that has ended
        table[i, 0] = pages.pop()
        refs[int(table[i, 0])] = 1
        lens[i] = r.randrange(1, PAGE + 1)
    shape = (len(refs), PAGE, case["heads_k"], case["dim"])
    as_int = lambda v: torch.as_tensor(v, dtype=torch.int32).to(DEVICE)  # noqa: E731
    children = list(range(case["parents"], rows))
    return {"path": "fork", "k_cache": normal(*shape), "v_cache": normal(*shape), "table": as_int(table),
            "lens": as_int(lens), "refs": as_int(refs), "children": as_int(children),
            "parents": as_int([i // kids for i in range(len(children))])}


def _prepare_compact(case, normal):
    r = random.Random(case["lengths"] + 1)
    pages = list(range(case["pages"]))
    r.shuffle(pages)
    common = [pages.pop() for _ in range(case["shared"])]
    table = torch.full((case["rows"], case["per_row"] + 2), -1, dtype=torch.int32)
    refs = torch.zeros(case["pages"], dtype=torch.int32)
    for i in range(case["rows"]):
        row = common + [pages.pop() for _ in range(case["per_row"] - case["shared"])]
        table[i, : len(row)] = torch.tensor(row, dtype=torch.int32)
        refs[row] += 1
    shape = (case["pages"], PAGE, case["heads_k"], case["dim"])
    return {"path": "compact", "k_cache": normal(*shape), "v_cache": normal(*shape), "table": table.to(DEVICE),
            "refs": refs.to(DEVICE)}


# ---------------------------------------------------------------------------
# One pass.


def run(state):
    path = state["path"]
    if own:
        return _run_own(_interface(), path, state)
    if path == "fork":
        return _plain_fork(state)
    if path == "compact":
        return _plain_compact(state)
    if path == "cache":
        return _plain_cache(state)
    if path == "varlen":
        return _plain_varlen(state)
    with torch.no_grad():
        return _plain_dense(state)


def _run_own(fai, path, s):
    if path == "fork":
        fai.flash_attn_kvcache_free(s["table"], s["lens"], s["refs"], s["children"], validate=False)
        fai.flash_attn_kvcache_fork(s["k_cache"], s["v_cache"], s["table"], s["lens"], s["refs"], s["parents"],
                                    s["children"], validate=False)
        fai.flash_attn_kvcache_alloc(s["table"], s["lens"], s["refs"], 1, PAGE, validate=False)
        return {name: s[name] for name in ("k_cache", "v_cache", "table", "lens", "refs")}
    if path == "compact":
        table, refs, used = fai.flash_attn_kvcache_compact(s["k_cache"], s["v_cache"], s["table"], s["refs"])
        return {"k_cache": s["k_cache"], "v_cache": s["v_cache"], "table": table, "refs": refs, "used": used}
    if path == "cache":
        out = fai.flash_diff_attn_with_kvcache(
            s["q"], s["k_cache"], s["v_cache"], s["lam"], s["k"], s["v"], cache_seqlens=s["lens"],
            cache_batch_idx=s["index"], block_table=s["table"], causal=True, validate=False)
        return {"out": out, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    if path == "prompt":
        with torch.no_grad():
            return {"out": fai.flash_diff_attn_func(s["q"], s["k"], s["v"], s["lam"], causal=s["causal"])}
    if path == "varlen":
        out = fai.flash_diff_attn_varlen_func(s["q"], s["k"], s["v"], s["lam"], s["cu"], s["cu"], s["longest"],
                                              s["longest"], causal=s["causal"])
    else:
        out = fai.flash_diff_attn_func(s["q"], s["k"], s["v"], s["lam"], causal=s["causal"])
    dq, dk, dv, dlam = torch.autograd.grad(out, (s["q"], s["k"], s["v"], s["lam"]), s["dout"])
    return {"out": out, "dq": dq, "dk": dk, "dv": dv, "dlam": dlam}


# ---------------------------------------------------------------------------
# The plain forms.


def _grouped(x, heads_k):
    """[b, s, heads, c] in 32 bits as [b, heads_k, group, s, c]."""
    b, s, h, c = x.shape
    return x.float().reshape(b, s, heads_k, h // heads_k, c).permute(0, 2, 3, 1, 4)


def _ungrouped(x):
    b, hk, g, s, c = x.shape
    return x.permute(0, 3, 1, 2, 4).reshape(b, s, hk * g, c)


def _by_row(lam, b, s, h, heads_k):
    """lam as [b, heads_k, group, s, 1]."""
    full = lam.float().expand(b, s, h)
    return _grouped(full[..., None], heads_k)


def _softmax(scores, visible):
    scores = torch.where(visible, scores, float("-inf"))
    top = scores.amax(-1, keepdim=True)
    e = torch.exp(scores - torch.where(top == float("-inf"), 0.0, top))
    total = e.sum(-1, keepdim=True)
    return e / torch.where(total > 0, total, 1.0)


def _product(a, b):
    """[b, hk, g, m, c] times [b, hk, c, n] for every head of a group."""
    n, hk, g, m, c = a.shape
    return torch.matmul(a.reshape(n, hk, g * m, c), b).reshape(n, hk, g, m, b.shape[-1])


def _maps(q, k, scale, visible):
    """Both maps of grouped q [b, hk, g, sq, dim] against k [b, hk, sk, dim]."""
    c = q.shape[-1] // 2
    one = _softmax(_product(q[..., :c], k[..., :c].transpose(-1, -2)) * scale, visible)
    two = _softmax(_product(q[..., c:], k[..., c:].transpose(-1, -2)) * scale, visible)
    return one, two


def _flat(x):
    b, hk, g, s, c = x.shape
    return x.reshape(b, hk, g * s, c)


def _gradients(q, k, v, lam, dout, one, two, scale):
    """Gradients of grouped q, of k and v, and of every row's lam, from the two maps."""
    c = q.shape[-1] // 2
    dp = _product(dout, v.transpose(-1, -2))
    dv = torch.matmul(_flat(one - lam * two).transpose(-1, -2), _flat(dout))
    d_two = (two * dp).sum(-1, keepdim=True)
    ds_one = one * (dp - (one * dp).sum(-1, keepdim=True)) * scale
    ds_two = two * (dp - d_two) * (-scale * lam)
    dq = torch.cat([_product(ds_one, k[..., :c]), _product(ds_two, k[..., c:])], -1)
    dk = torch.cat([torch.matmul(_flat(ds_one).transpose(-1, -2), _flat(q[..., :c])),
                    torch.matmul(_flat(ds_two).transpose(-1, -2), _flat(q[..., c:]))], -1)
    return dq, dk, dv, -d_two


def _like(dlam, lam):
    """The gradient of every row's lam, [b, s, h], summed to lam's own shape."""
    if lam.dim() == 0:
        return dlam.double().sum().float()
    if lam.dim() == 1:
        return dlam.double().sum((0, 1)).float()
    return dlam


def _causal(sq, sk, device):
    return torch.arange(sk, device=device) <= torch.arange(sq, device=device)[:, None] + (sk - sq)


def _plain_dense(s):
    q, k, v, lam = s["q"], s["k"], s["v"], s["lam"]
    b, sq, h, dim = q.shape
    sk, hk = k.shape[1], k.shape[2]
    qg, kg, vg = _grouped(q, hk), _grouped(k, hk)[:, :, 0], _grouped(v, hk)[:, :, 0]
    row = _by_row(lam, b, sq, h, hk)
    visible = _causal(sq, sk, q.device) if s["causal"] else torch.ones(sq, sk, dtype=torch.bool, device=q.device)
    one, two = _maps(qg, kg, s["scale"], visible)
    got = {"out": _ungrouped(_product(one - row * two, vg)).to(q.dtype)}
    if s["path"] == "prompt":
        return got
    dq, dk, dv, dlam = _gradients(qg, kg, vg, row, _grouped(s["dout"], hk), one, two, s["scale"])
    got["dq"] = _ungrouped(dq).to(q.dtype)
    got["dk"], got["dv"] = (x.transpose(1, 2).to(q.dtype) for x in (dk, dv))
    got["dlam"] = _like(_ungrouped(dlam)[..., 0], lam)
    return got


def _plain_varlen(s):
    """The packed rows in a padded batch and back."""
    with torch.no_grad():
        q, k, v, lam, cu, n = s["q"], s["k"], s["v"], s["lam"], s["cu"].long(), s["longest"]
        hk, h = k.shape[1], q.shape[1]
        lens = cu[1:] - cu[:-1]
        at = torch.arange(n, device=q.device)
        real = at < lens[:, None]
        rows = torch.where(real, cu[:-1, None] + at, 0)
        b = lens.numel()
        pad = lambda x: torch.where(real[..., None, None], x.float()[rows], 0.0)  # noqa: E731
        qg, dog = _grouped(pad(q), hk), _grouped(pad(s["dout"]), hk)
        kg, vg = _grouped(pad(k), hk)[:, :, 0], _grouped(pad(v), hk)[:, :, 0]
        row = _by_row(lam[rows] if lam.dim() == 2 else lam, b, n, h, hk)
        visible = real[:, None, :] & real[:, :, None]
        if s["causal"]:
            visible = visible & (at <= at[:, None])
        one, two = _maps(qg, kg, s["scale"], visible[:, None, None])
        dq, dk, dv, dlam = _gradients(qg, kg, vg, row, dog, one, two, s["scale"])
        packed = lambda x: x[real]  # noqa: E731
        got = {"out": packed(_ungrouped(_product(one - row * two, vg))).to(q.dtype),
               "dq": packed(_ungrouped(dq)).to(q.dtype)}
        got["dk"], got["dv"] = (packed(x.transpose(1, 2)).to(q.dtype) for x in (dk, dv))
        dlam = packed(_ungrouped(dlam)[..., 0])
        got["dlam"] = dlam if lam.dim() == 2 else _like(dlam[None], lam)
        return got


def _plain_cache(s):
    q, k, v, lens = s["q"], s["k"], s["v"], s["lens"].long()
    b, n, h, dim = q.shape
    hk = k.shape[2]
    new = lens[:, None] + torch.arange(n, device=q.device)  # positions of the new tokens
    if s["table"] is not None:
        pages = s["table"].long()
        capacity = pages.shape[1] * PAGE
        place = (pages.gather(1, new // PAGE), new % PAGE)
    else:
        rows = torch.arange(b, device=q.device) if s["index"] is None else s["index"].long()
        capacity = s["k_cache"].shape[1]
        place = (rows[:, None].expand(-1, n), new)
    s["k_cache"][place], s["v_cache"][place] = k, v

    def tokens(cache):
        if s["table"] is not None:
            return cache[pages.clamp_min(0)].reshape(b, capacity, hk, dim).float().transpose(1, 2)
        return cache[rows].float().transpose(1, 2)

    row = _by_row(s["lam"], b, n, h, hk)
    visible = torch.arange(capacity, device=q.device) <= new[..., None]
    one, two = _maps(_grouped(q, hk), tokens(s["k_cache"]), s["scale"], visible[:, None, None])
    out = _ungrouped(_product(one - row * two, tokens(s["v_cache"]))).to(q.dtype)
    return {"out": out, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _plain_fork(s):
    table, lens, refs, kids, parents = s["table"], s["lens"], s["refs"], s["children"].long(), s["parents"].long()
    width = table.shape[1]
    # The children's rows end: their pages are given back.
    held = table[kids]
    refs.sub_(torch.bincount(held[held >= 0].long(), minlength=refs.numel()).int())
    table[kids], lens[kids] = -1, 0
    # Each child shares its parent's full pages and has a copy of the used part of the last one.
    length = lens[parents].long()
    column = torch.arange(width, device=table.device)
    full = column < (length // PAGE)[:, None]
    part = (length % PAGE > 0) & (length // PAGE < width)
    rows = torch.where(full, table[parents], -1)
    refs.add_(torch.bincount(rows[rows >= 0].long(), minlength=refs.numel()).int())
    copies = part.nonzero()[:, 0]
    fresh = (refs == 0).nonzero()[: copies.numel(), 0]
    last = (length // PAGE)[copies]
    old = table[parents[copies], last].long()
    rows[copies, last] = fresh.int()
    refs[fresh] = 1
    table[kids], lens[kids] = rows, length.int()
    used = torch.arange(PAGE, device=table.device) < (length % PAGE)[copies][:, None]
    for cache in (s["k_cache"], s["v_cache"]):
        cache[fresh] = torch.where(used[..., None, None], cache[old], cache[fresh])
    # Every row gets a page where its next token needs one.
    page = lens.long() // PAGE
    rows = ((page < width) & (table.gather(1, page.clamp_max(width - 1)[:, None])[:, 0] < 0)).nonzero()[:, 0]
    fresh = (refs == 0).nonzero()[: rows.numel(), 0]
    table[rows, page[rows]] = fresh.int()
    refs[fresh] = 1
    return {name: s[name] for name in ("k_cache", "v_cache", "table", "lens", "refs")}


def _plain_compact(s):
    table, refs = s["table"], s["refs"]
    used = refs > 0
    count = used.sum()
    front = torch.arange(refs.numel(), device=refs.device) < count
    holes, movers = (front & ~used).nonzero()[:, 0], (used & ~front).nonzero()[:, 0]
    place = torch.arange(refs.numel(), dtype=torch.int32, device=refs.device)
    place[movers] = holes.int()
    new_refs = refs.clone()
    new_refs[holes], new_refs[movers] = refs[movers], 0
    for cache in (s["k_cache"], s["v_cache"]):
        cache[holes] = cache[movers]
    new_table = torch.where(table >= 0, place[table.clamp_min(0).long()], table)
    return {"k_cache": s["k_cache"], "v_cache": s["v_cache"], "table": new_table, "refs": new_refs,
            "used": count.int().reshape(1)}


# ---------------------------------------------------------------------------
# From the definition, in 64 bits.


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        if case["path"] == "fork":
            return _exact_fork(s)
        if case["path"] == "compact":
            return _exact_compact(s)
        if case["path"] == "cache":
            return _exact_cache(s)
        q, k, v, lam = s["q"], s["k"], s["v"], s["lam"].double()
        grad = case["path"] != "prompt"
        got = {"out": torch.empty(q.shape, dtype=torch.float64, device=DEVICE)}
        if grad:
            for name, x in (("dq", q), ("dk", k), ("dv", v)):
                got[name] = torch.zeros(x.shape, dtype=torch.float64, device=DEVICE)
            got["dlam"] = torch.zeros_like(lam)
        ends = s["cu"].tolist() if case["path"] == "varlen" else None
        for b in range(len(ends) - 1 if ends else q.shape[0]):
            at = slice(ends[b], ends[b + 1]) if ends else b
            for h in range(case["heads"]):
                j = h // (case["heads"] // case["heads_k"])
                row = lam if lam.dim() == 0 else lam[h] if lam.dim() == 1 else lam[at][:, h : h + 1]
                dout = s["dout"][at][:, h].double() if grad else None
                o, g = _exact_head(q[at][:, h].double(), k[at][:, j].double(), v[at][:, j].double(), row, s["scale"],
                                   s["causal"], dout)
                got["out"][at][:, h] = o
                if grad:
                    got["dq"][at][:, h] = g[0]
                    got["dk"][at][:, j] += g[1]
                    got["dv"][at][:, j] += g[2]
                    if lam.dim() == 0:
                        got["dlam"] += g[3].sum()
                    elif lam.dim() == 1:
                        got["dlam"][h] += g[3].sum()
                    else:
                        got["dlam"][at][:, h] = g[3]
        return got


def _exact_head(q, k, v, lam, scale, causal, dout=None):
    """One head of one sequence: o, and (dq, dk, dv, dlam of each row) when dout is given."""
    sq, sk, c = q.shape[0], k.shape[0], q.shape[1] // 2
    hidden = torch.zeros(sq, sk, dtype=torch.bool, device=q.device)
    if causal:
        hidden = torch.ones(sq, sk, dtype=torch.bool, device=q.device).triu(sk - sq + 1)
    weights = []
    for m in (0, 1):
        x = (q[:, m * c : m * c + c] @ k[:, m * c : m * c + c].T * scale).masked_fill(hidden, -math.inf)
        x = (x - x.max(1, keepdim=True).values.nan_to_num(neginf=0.0)).exp()
        weights.append(x / x.sum(1, keepdim=True).clamp_min(1e-300))
    a, w = weights
    o = (a - lam * w) @ v
    if dout is None:
        return o, None
    d = dout @ v.T
    da = a * (d - (a * d).sum(1, keepdim=True))
    mean = (w * d).sum(1, keepdim=True)
    dw = w * (mean - d) * lam
    dq = torch.cat((da @ k[:, :c], dw @ k[:, c:]), 1) * scale
    dk = torch.cat((da.T @ q[:, :c], dw.T @ q[:, c:]), 1) * scale
    return o, (dq, dk, (a - lam * w).T @ dout, -mean[:, 0])


def _exact_cache(s):
    b, n, h, dim = s["q"].shape
    hk = s["k"].shape[2]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device=DEVICE)
    lam = s["lam"].double()
    for i, length in enumerate(s["lens"].tolist()):
        end = length + n
        caches = []
        for cache, new in ((s["k_cache"], s["k"]), (s["v_cache"], s["v"])):
            if s["table"] is None:
                line = cache[i if s["index"] is None else int(s["index"][i])]
                line[length:end] = new[i]
                caches.append(line[:end])
                continue
            pages = s["table"][i].tolist()
            for j in range(length // PAGE, -(-end // PAGE)):
                first, last = max(length, j * PAGE), min(end, (j + 1) * PAGE)
                cache[pages[j], first - j * PAGE : last - j * PAGE] = new[i, first - length : last - length]
            caches.append(torch.cat([cache[p] for p in pages[: -(-end // PAGE)]])[:end])
        for head in range(h):
            j = head // (h // hk)
            row = lam if lam.dim() == 0 else lam[head] if lam.dim() == 1 else lam[i, :, head, None]
            out[i, :, head] = _exact_head(s["q"][i, :, head].double(), caches[0][:, j].double(),
                                          caches[1][:, j].double(), row, s["scale"], True)[0]
    return {"out": out, "k_cache": s["k_cache"].double(), "v_cache": s["v_cache"].double()}


def _exact_fork(s):
    table, lens, refs = s["table"].tolist(), s["lens"].tolist(), s["refs"].tolist()
    parents, kids = s["parents"].tolist(), s["children"].tolist()
    for c in kids:
        for page in table[c]:
            if page >= 0:
                refs[page] -= 1
        table[c], lens[c] = [-1] * len(table[c]), 0
    for p, c in zip(parents, kids):
        for j in range(lens[p] // PAGE):
            table[c][j] = table[p][j]
            refs[table[p][j]] += 1
        lens[c] = lens[p]
    for p, c in zip(parents, kids):
        j, rest = divmod(lens[p], PAGE)
        if rest:
            page = refs.index(0)
            refs[page], table[c][j] = 1, page
            for cache in (s["k_cache"], s["v_cache"]):
                cache[page, :rest] = cache[table[p][j], :rest]
    for row, length in zip(table, lens):
        j = length // PAGE
        if row[j] < 0:
            row[j] = refs.index(0)
            refs[row[j]] = 1
    whole = lambda v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    return {"k_cache": s["k_cache"].double(), "v_cache": s["v_cache"].double(), "table": whole(table),
            "lens": whole(lens), "refs": whole(refs)}


def _exact_compact(s):
    table, refs = s["table"].tolist(), s["refs"].tolist()
    count = sum(n > 0 for n in refs)
    free = [p for p in range(count) if not refs[p]]
    moved = dict(zip([p for p in range(count, len(refs)) if refs[p]], free))
    for old, new in moved.items():
        for cache in (s["k_cache"], s["v_cache"]):
            cache[new] = cache[old]
        refs[new], refs[old] = refs[old], 0
    table = [[moved.get(p, p) for p in row] for row in table]
    whole = lambda v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    return {"k_cache": s["k_cache"].double(), "v_cache": s["v_cache"].double(), "table": whole(table),
            "refs": whole(refs), "used": whole([count])}
