"""The attention half of a decoder layer on an 8-bit paged cache: what is measured.

Four operators over real work: rotary positions (and their inverse, the gradient), appending new
keys and values to a cache of int8 codes with one scale for each page and head, attention over that
cache (one token, a few tokens and whole prompts per sequence), and the page bookkeeping between steps
(fork / free / reserve, compact). Where ``own`` is false, ``run`` computes them from elementary torch
operations in 32 bits; where it is true, with the framework's kernels.

Conventions shared by both: ``tables`` int32 [sequences, width] holds page numbers (-1: none),
``lengths`` int32 the tokens that a sequence holds with the step's new ones, ``starts`` int32
[sequences + 1] the rows of the step's new tokens; the j-th of a sequence's n new tokens stands at
position lengths - n + j. A sequence of length 0 is an idle slot of the batch.
"""
import math
import random

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


# ------------------------------------------------------------------------------------- the cases
def listed():
    return [
        # queries of one decode batch (64 heads of d_model 8192): a launch's latency
        {"name": "rotary-decode-32", "op": "rotary", "tokens": 32, "heads": 64, "dim": 128, "rot": 128,
         "interleaved": False, "inverse": False, "packed": False, "dtype": "f16"},
        # gradient of a long batch's queries, rotated on part of the head, inside a packed q/k/v row
        {"name": "rotary-back-16384", "op": "rotary", "tokens": 16384, "heads": 32, "dim": 128, "rot": 64,
         "interleaved": True, "inverse": True, "packed": True, "dtype": "bf16"},
        # one decode step of 64 sequences: rotate q and k, grow the open blocks' scales, write one token each
        {"name": "append-decode-64", "op": "append", "seqs": 64, "kv_heads": 8, "heads": 64, "dim": 128, "page": 64,
         "longest": 4096, "chunk": 1, "interleaved": False, "dtype": "f16"},
        # ragged prompt chunks of a prefill batch
        {"name": "append-chunks-8k", "op": "append", "seqs": 12, "kv_heads": 8, "heads": 32, "dim": 128, "page": 64,
         "longest": 6000, "chunk": 1365, "interleaved": True, "dtype": "bf16"},
        # one user, short context, small pages: latency
        {"name": "decode-1x777", "op": "attend", "seqs": 1, "kv_heads": 8, "group": 4, "dim": 128, "page": 16,
         "longest": 777, "chunk": 0, "window": 0, "dtype": "f16"},
        # a serving batch with contexts from a few tokens to 32k, one slot idle
        {"name": "decode-24x32k", "op": "attend", "seqs": 24, "kv_heads": 8, "group": 8, "dim": 128, "page": 64,
         "longest": 32768, "chunk": 0, "window": 0, "dtype": "bf16"},
        # a 2048-token prompt chunk on top of earlier context, beside shorter ones
        {"name": "chunk-3x2048", "op": "attend", "seqs": 3, "kv_heads": 8, "group": 8, "dim": 128, "page": 64,
         "longest": 6144, "chunk": 2048, "window": 0, "dtype": "f16"},
        # a whole long prompt
        {"name": "prefill-8192", "op": "attend", "seqs": 1, "kv_heads": 8, "group": 4, "dim": 128, "page": 128,
         "longest": 8192, "chunk": 8192, "window": 0, "dtype": "bf16"},
        # four samples for each of 16 prompts: shared pages, copies of the open ones
        {"name": "fork-16-to-64", "op": "fork", "seqs": 16, "children": 64, "pages": 1024, "layers": 2, "kv_heads": 8,
         "dim": 128, "page": 64, "longest": 2048},
        # reordered beams of a large batch over a deep stack
        {"name": "fork-64-to-256", "op": "fork", "seqs": 64, "children": 256, "pages": 4096, "layers": 8, "kv_heads": 8,
         "dim": 128, "page": 32, "longest": 1500},
        # a small pool after its requests thinned out
        {"name": "compact-300", "op": "compact", "seqs": 20, "pages": 300, "used": 130, "moved": 41, "layers": 2,
         "kv_heads": 8, "dim": 128, "page": 16},
        # a large pool
        {"name": "compact-4096", "op": "compact", "seqs": 128, "pages": 4096, "used": 2048, "moved": 700, "layers": 4,
         "kv_heads": 8, "dim": 128, "page": 64},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw(rng):
    op = rng.choice(["rotary", "append", "attend", "attend", "attend", "fork", "compact"])
    dtype = rng.choice(["f16", "bf16"])
    if op == "rotary":
        dim = rng.choice([64, 80, 96, 128, 256])
        return {"op": op, "tokens": _log(rng, 1, 16384), "heads": rng.choice([1, 5, 8, 32, 40, 64]), "dim": dim,
                "rot": rng.choice([dim, dim // 2]), "interleaved": rng.random() < 0.5, "inverse": rng.random() < 0.3,
                "packed": rng.random() < 0.5, "dtype": rng.choice(["f16", "bf16", "f32"])}
    kv_heads, dim, page = rng.choice([1, 2, 5, 8, 16]), rng.choice([64, 128, 256]), rng.choice([16, 32, 64, 128])
    if op == "append":
        group = rng.choice([1, 4, 5, 8])
        return {"op": op, "seqs": _log(rng, 1, 128), "kv_heads": kv_heads, "heads": kv_heads * group, "dim": dim,
                "page": page, "longest": _log(rng, 16, 8192), "chunk": rng.choice([1, 1, _log(rng, 2, 1500)]),
                "interleaved": rng.random() < 0.5, "dtype": dtype}
    if op == "attend":
        longest = _log(rng, 20, 40000)
        return {"op": op, "seqs": _log(rng, 1, 64), "kv_heads": kv_heads, "group": rng.choice([1, 2, 4, 5, 8, 16]),
                "dim": dim, "page": page, "longest": longest,
                "chunk": rng.choice([0, 0, rng.randint(2, 8), min(longest, _log(rng, 16, 8192))]),
                "window": rng.choice([0, 0, 0, 1024]), "dtype": dtype}
    if op == "fork":
        seqs = _log(rng, 1, 64)
        children, longest = _log(rng, seqs, 256), _log(rng, 40, 4000)
        return {"op": op, "seqs": seqs, "children": children,
                "pages": seqs * -(-longest // page) + children * 3 + rng.randint(1, 200), "layers": rng.randint(1, 8),
                "kv_heads": kv_heads, "dim": dim, "page": page, "longest": longest}
    pages = _log(rng, 40, 4096)
    used = max(2, int(pages * rng.uniform(0.1, 0.9)))
    return {"op": op, "seqs": rng.randint(1, min(used, 128)), "pages": pages, "used": used,
            "moved": rng.randint(1, max(1, min(used - 1, pages - used))), "layers": rng.randint(1, 4),
            "kv_heads": kv_heads, "dim": dim, "page": page}


def draw(rng):
    top = {}
    for c in listed():
        w = work(c)
        top[c["op"]] = [max(a, b) for a, b in zip(top.get(c["op"], (0, 0)), (w["bytes"], w["flops"]))]
    while True:
        c = _draw(rng)
        w = work(c)
        if w["bytes"] > top[c["op"]][0] or w["flops"] > top[c["op"]][1]:
            continue
        if c["op"] == "attend":  # the plain form pads to the longest sequence and holds every score
            new, lengths = _attend_shape(c)
            rows = c["seqs"] * max(new) * c["kv_heads"] * c["group"]
            if rows * max(lengths) > 3e9 or c["seqs"] * max(lengths) * c["kv_heads"] * c["dim"] > 1.7e9:
                continue
        return c


# --------------------------------------------------------- shapes that follow from a case's numbers
def _rng(case, salt):
    return random.Random("%s %s" % (salt, sorted((k, v) for k, v in case.items() if k != "name")))


def _append_shape(case):
    """New tokens and lengths of each sequence: every length over the range up to the longest."""
    r, B = _rng(case, "append"), case["seqs"]
    if case["chunk"] == 1:
        new = [1] * B
    else:
        new = [r.randint(1, case["chunk"]) for _ in range(B)]
        new[0] = case["chunk"]
    held = [_log(r, 1, case["longest"]) for _ in range(B)]
    held[-1] = 0  # a new sequence
    return new, [a + b for a, b in zip(new, held)]


def _attend_shape(case):
    """chunk 0: one token for each sequence (no starts); else 1 .. chunk new tokens each."""
    r, B, longest, chunk = _rng(case, "attend"), case["seqs"], case["longest"], case["chunk"]
    new = [1] * B if chunk == 0 else [r.randint(1, chunk) for _ in range(B)]
    if chunk:
        new[0] = chunk
    lengths = [max(n, _log(r, max(1, longest // 64), longest)) for n in new]
    lengths[0] = longest
    if B >= 4 and chunk == 0:
        lengths[1] = 0  # an idle slot
        lengths[2] = 1
    return new, lengths


def _fork_shape(case):
    """Lengths (every one with an open last page), parents and room for new tokens of each child."""
    r, P = _rng(case, "fork"), case["page"]
    lengths = []
    for _ in range(case["seqs"]):
        n = r.randint(max(1, case["longest"] // 4), case["longest"])
        lengths.append(n - 1 if n % P == 0 else n)
    parents = [i % case["seqs"] for i in range(case["children"])]
    r.shuffle(parents)
    if case["seqs"] > 2:  # one sequence ends, its place in the batch is empty
        drop = parents[0]
        parents = [-1 if p == drop else p for p in parents]
    extra = [r.choice([1, 1, 2]) for _ in parents]
    return lengths, parents, extra


def _compact_shape(case):
    """Pages of each sequence; `moved` of the used ones lie at or above `used`."""
    r, U = _rng(case, "compact"), case["used"]
    cuts = sorted(r.sample(range(1, U), case["seqs"] - 1)) if case["seqs"] > 1 else []
    counts = [b - a for a, b in zip([0] + cuts, cuts + [U])]
    lengths = [c * case["page"] - r.randint(0, case["page"] - 1) for c in counts]
    return counts, lengths


def _page_bytes(case):
    return 2 * case["kv_heads"] * (case["page"] * case["dim"] + 4)


def work(case):
    op = case["op"]
    if op == "rotary":
        size = 4 if case["dtype"] == "f32" else 2
        n = case["tokens"] * case["heads"] * case["dim"]
        return {"bytes": 2 * n * size + case["tokens"] * (4 + 4 * case["rot"]),
                "flops": 3 * case["tokens"] * case["heads"] * case["rot"]}
    if op == "append":
        new, lengths = _append_shape(case)
        T, row, P = sum(new), case["kv_heads"] * case["dim"], case["page"]
        seen = sum(a - (a - n) // P * P for a, n in zip(lengths, new))  # tokens of the blocks that change
        pages = sum(-(-a // P) - (a - n) // P for a, n in zip(lengths, new))
        return {"bytes": T * (2 * row * 2 + 2 * case["heads"] * case["dim"] * 2 + 4 * case["dim"]) + 2 * T * row
                + (seen - T) * 2 * row + pages * case["kv_heads"] * 16 + seen * 2 * row * 5,
                "flops": 8 * T * row + 3 * T * case["heads"] * case["dim"]}
    if op == "attend":
        new, lengths = _attend_shape(case)
        pairs, keys, w = 0, 0, case["window"]
        for n, a in zip(new, lengths):
            if a == 0:
                continue
            first = a - n
            if w:
                pairs += sum(min(first + i + 1, w) for i in range(n))
                keys += a - max(0, first + 1 - w)
            else:
                pairs += n * first + n * (n + 1) // 2
                keys += a
        H, D = case["kv_heads"] * case["group"], case["dim"]
        return {"bytes": 2 * keys * case["kv_heads"] * D + 4 * sum(new) * H * D + keys // case["page"] * (8 * case["kv_heads"] + 4),
                "flops": 4 * pairs * H * D}
    if op == "fork":
        lengths, parents, extra = _fork_shape(case)
        P = case["page"]
        kept = {p for p in parents if p >= 0}
        copies = sum(p >= 0 for p in parents) - len(kept)
        entries = sum(-(-lengths[p] // P) for p in kept)
        out = sum(-(-((lengths[p] if p >= 0 else 0) + e) // P) for p, e in zip(parents, extra))
        return {"bytes": 2 * copies * case["layers"] * _page_bytes(case) + 4 * (entries + out + 3 * len(parents)), "flops": 0}
    return {"bytes": 2 * case["moved"] * case["layers"] * _page_bytes(case) + 8 * case["used"] + 4 * case["seqs"], "flops": 0}


# ------------------------------------------------------------------------------------------- inputs
def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _rows(new):
    at = [0]
    for n in new:
        at.append(at[-1] + n)
    return at


def _cos_sin(positions, rot):
    f = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot)
    a = torch.arange(positions, dtype=torch.float64, device="cuda")[:, None] * f
    return torch.cat([a.cos(), a.sin()], 1).float()


def _pool(case, layers, pages, g, live=None):
    """Codes of normally distributed values; pages that no sequence holds have NaN scales."""
    H, P, D = case["kv_heads"], case["page"], case["dim"]
    out = []
    for _ in range(2):
        codes = torch.empty(layers, pages, H, P, D, dtype=torch.int8, device="cuda")
        flat = codes.view(-1)
        for at in range(0, flat.numel(), 1 << 28):
            part = flat[at:at + (1 << 28)]
            part.copy_((torch.randn(part.numel(), device="cuda", generator=g) * 38).round_().clamp_(-127, 127))
        scale = 0.02 + 0.02 * torch.rand(layers, pages, H, device="cuda", generator=g)
        if live is not None:
            dead = torch.ones(pages, dtype=torch.bool, device="cuda")
            dead[live.long()] = False
            scale[:, dead] = float("nan")
        out += [codes, scale]
    return {"k_codes": out[0], "k_scale": out[1], "v_codes": out[2], "v_scale": out[3]}


def _tables(counts, width, pages, g):
    """Page numbers of each sequence, drawn without order from the pool."""
    order = torch.randperm(pages, device="cuda", generator=g).int()
    t = torch.full((len(counts), width), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(counts):
        t[b, :n] = order[at:at + n]
        at += n
    return t, order[:at]


def _handle(case, s, layers, pages, seqs):
    if own:
        from ffn_residual_mesh_b200.kvcache import PagedKvCache
        s["cache"] = PagedKvCache(layers, pages, case["kv_heads"], case["dim"], page_tokens=case["page"], max_seqs=seqs,
                                  buffers=(s["k_codes"], s["v_codes"], s["k_scale"], s["v_scale"]))


def _rope(case, s, cos_sin):
    s["cos_sin"] = cos_sin
    if own:
        from ffn_residual_mesh_b200.kvcache import RotaryTable
        s["rope"] = RotaryTable.from_tensor(cos_sin, interleaved=case["interleaved"])


def _randn(shape, g, dtype):
    return torch.randn(shape, device="cuda", generator=g).to(dtype)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op, s = case["op"], {"case": case}
    if op == "rotary":
        T, H, D, dtype = case["tokens"], case["heads"], case["dim"], DTYPES[case["dtype"]]
        x = _randn((T, H + 2 if case["packed"] else H, D), g, dtype)
        s["x"] = x[:, :H]  # in a packed row, keys and values of one head follow
        most = max(4096, T)
        s["positions"] = torch.randint(0, most, (T,), device="cuda", generator=g).int()
        _rope(case, s, _cos_sin(most, case["rot"]))
        return s
    if op == "append":
        new, lengths = _append_shape(case)
        H, Hk, D, P, B = case["heads"], case["kv_heads"], case["dim"], case["page"], case["seqs"]
        counts = [-(-a // P) for a in lengths]
        pages = sum(counts) + 7
        s["tables"], live = _tables(counts, max(counts) + 1, pages, g)
        s.update(_pool(case, 1, pages, g, live))
        for name in ("k_scale", "v_scale"):  # smaller than the new tokens often ask for: some blocks grow
            s[name].mul_(0.8)
        at = _rows(new)
        qkv = _randn((at[-1], H + 2 * Hk, D), g, DTYPES[case["dtype"]])
        s["q"], s["k"], s["v"] = qkv[:, :H], qkv[:, H:H + Hk], qkv[:, H + Hk:]
        s["lengths"], s["starts"] = _ints(lengths), _ints(at)
        seen = [a - (a - n) // P * P for a, n in zip(lengths, new)]
        s["seen"], s["rows"] = _ints(_rows(seen)), sum(seen)
        _rope(case, s, _cos_sin(max(lengths), D))
        _handle(case, s, 1, pages, B)
        return s
    if op == "attend":
        new, lengths = _attend_shape(case)
        counts = [-(-a // case["page"]) for a in lengths]
        pages = sum(counts) + 5
        s["tables"], live = _tables(counts, max(counts) + 1, pages, g)
        s.update(_pool(case, 1, pages, g, live))
        at = _rows(new)
        s["q"] = _randn((at[-1], case["kv_heads"] * case["group"], case["dim"]), g, DTYPES[case["dtype"]])
        s["lengths"] = _ints(lengths)
        s["starts"] = _ints(at) if case["chunk"] else None
        s["most_new"], s["longest"] = max(new), max(lengths)
        _handle(case, s, 1, pages, case["seqs"])
        return s
    if op == "fork":
        lengths, parents, extra = _fork_shape(case)
        counts = [-(-a // case["page"]) for a in lengths]
        width = -(-(case["longest"] + 2) // case["page"]) + 1
        s["tables"], _ = _tables(counts, width, case["pages"], g)
        s.update(_pool(case, case["layers"], case["pages"], g))
        s["lengths"], s["parents"], s["extra"] = _ints(lengths), _ints(parents), _ints(extra)
        _handle(case, s, case["layers"], case["pages"], max(case["seqs"], case["children"]))
        return s
    counts, lengths = _compact_shape(case)
    U, m = case["used"], case["moved"]
    low = torch.randperm(U, device="cuda", generator=g)[:U - m]
    high = U + torch.randperm(case["pages"] - U, device="cuda", generator=g)[:m]
    order = torch.cat([low, high])[torch.randperm(U, device="cuda", generator=g)].int()
    t = torch.full((case["seqs"], max(counts)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(counts):
        t[b, :n] = order[at:at + n]
        at += n
    s["tables"], s["lengths"] = t, _ints(lengths)
    s.update(_pool(case, case["layers"], case["pages"], g))
    _handle(case, s, case["layers"], case["pages"], case["seqs"])
    return s


# --------------------------------------------------------------------------------------- plain forms
def _rotate(x, rows, interleaved, inverse=False):
    """x [T, H, D] in 32 bits, rows [T, R] of the cos | sin table."""
    R = rows.shape[1]
    c, s = rows[:, None, :R // 2], rows[:, None, R // 2:]
    if inverse:
        s = -s
    a, b = (x[..., 0:R:2], x[..., 1:R:2]) if interleaved else (x[..., :R // 2], x[..., R // 2:R])
    y, z = a * c - b * s, b * c + a * s
    out = x.clone()
    if interleaved:
        out[..., 0:R:2], out[..., 1:R:2] = y, z
    else:
        out[..., :R // 2], out[..., R // 2:R] = y, z
    return out


def _places(starts, lengths, tables, P, total):
    """Sequence, position, page and slot of each of `total` rows."""
    rows = torch.arange(total, device="cuda", dtype=torch.int32)
    seq = torch.searchsorted(starts, rows, right=True).long() - 1
    pos = (rows - starts[seq + 1] + lengths[seq]).long()
    return seq, pos, tables[seq, pos // P].long(), pos % P


def _plain_append(s):
    case, P = s["case"], s["case"]["page"]
    seq, pos, page, slot = _places(s["starts"], s["lengths"], s["tables"], P, s["k"].shape[0])
    rows = s["cos_sin"][pos]
    q = _rotate(s["q"].float(), rows, case["interleaved"]).to(s["q"].dtype)
    k, v = _rotate(s["k"].float(), rows, case["interleaved"]), s["v"].float()
    held = s["lengths"] - (s["starts"][1:] - s["starts"][:-1])  # before the step
    has = held % P > 0
    open_page = s["tables"].gather(1, (held // P).long()[:, None])[:, 0].long()[has]
    open_slots = torch.arange(P, device="cuda") < (held % P)[has][:, None]
    top = torch.tensor(127.0, device="cuda")
    back = torch.searchsorted(s["seen"], torch.arange(s["rows"], device="cuda", dtype=torch.int32), right=True).long() - 1
    _, _, read_page, read_slot = _places(s["seen"], s["lengths"], s["tables"], P, s["rows"])
    out = [q]
    for x, codes, scale in ((k, s["k_codes"][0], s["k_scale"][0]), (v, s["v_codes"][0], s["v_scale"][0])):
        most = torch.zeros_like(scale).index_reduce_(0, page, x.abs().amax(-1), "amax")
        before = torch.zeros_like(scale)
        before[open_page] = scale[open_page]
        fresh = torch.maximum(torch.maximum(before, most / top), torch.full_like(scale, 1e-12))
        scale[page] = fresh[page]
        old = codes[open_page]
        grown = (old.float() * (before[open_page] / fresh[open_page])[..., None, None]).round()
        codes[open_page] = torch.where(open_slots[:, None, :, None], grown.to(torch.int8), old)
        codes[page, :, slot] = (x / fresh[page][..., None]).round().clamp(-127, 127).to(torch.int8)
        out.append(codes[read_page, :, read_slot].float() * scale[read_page][..., None])
    return out


def _plain_attend(s):
    case = s["case"]
    B, Hk, G, D, P = case["seqs"], case["kv_heads"], case["group"], case["dim"], case["page"]
    q, lengths, most, L = s["q"], s["lengths"], s["most_new"], s["longest"]
    W = -(-L // P)
    total = q.shape[0]
    starts = s["starts"] if s["starts"] is not None else torch.arange(B + 1, device="cuda", dtype=torch.int32)
    new = starts[1:] - starts[:-1]
    seq = torch.searchsorted(starts, torch.arange(total, device="cuda", dtype=torch.int32), right=True).long() - 1
    at = torch.arange(total, device="cuda") - starts[seq].long()
    padded = torch.zeros(B, most, Hk, G, D, device="cuda")
    padded[seq, at] = q.float().view(total, Hk, G, D)
    padded = padded.permute(0, 2, 1, 3, 4).reshape(B, Hk, most * G, D)
    table = s["tables"][:, :W].long().clamp(min=0)
    key = torch.arange(W * P, device="cuda")
    live = key < lengths[:, None]  # [B, keys]

    def values(codes, scale):
        x = codes[0][table].float() * scale[0][table][..., None, None]  # [B, W, Hk, P, D]
        x = x.permute(0, 2, 1, 3, 4).reshape(B, Hk, W * P, D)
        return x.masked_fill_(~live[:, None, :, None], 0.0)

    scores = padded @ values(s["k_codes"], s["k_scale"]).transpose(-1, -2)
    scores *= 1.0 / math.sqrt(D)
    pos = (lengths - new)[:, None] + torch.arange(most, device="cuda")  # [B, most]
    seen = live[:, None] & (key <= pos[..., None])
    if case["window"]:
        seen &= key > pos[..., None] - case["window"]
    scores.view(B, Hk, most, G, W * P).masked_fill_(~seen[:, None, :, None], float("-inf"))
    top = scores.amax(-1, keepdim=True)
    scores -= top.masked_fill_(top == float("-inf"), 0.0)
    scores.exp_()
    total_p = scores.sum(-1, keepdim=True)
    out = (scores @ values(s["v_codes"], s["v_scale"])) / total_p.masked_fill_(total_p == 0, 1.0)
    out = out.view(B, Hk, most, G, D).permute(0, 2, 1, 3, 4)
    return out[seq, at].reshape(total, Hk * G, D).to(q.dtype)


def _plain_fork(s):
    case, tables, P, N = s["case"], s["tables"], s["case"]["page"], s["case"]["pages"]
    parents, extra = s["parents"].long(), s["extra"]
    W = tables.shape[1]
    length = torch.where(parents >= 0, s["lengths"][parents.clamp(min=0)], 0)
    t = tables[parents.clamp(min=0)].long()
    col = torch.arange(W, device="cuda")
    full = (length // P).long()
    is_full = col < full[:, None]
    part = length % P > 0
    whole = torch.zeros(N, dtype=torch.bool, device="cuda")
    whole[t[is_full]] = True
    last = t.gather(1, full.clamp(max=W - 1)[:, None])[:, 0]
    child = torch.arange(len(parents), device="cuda")
    first = torch.full((N,), len(parents), device="cuda", dtype=torch.long)
    first.scatter_reduce_(0, last[part], child[part], "amin")
    keep = part & ~whole[last.clamp(min=0)] & (first[last.clamp(min=0)] == child)
    used = whole
    used[last[keep]] = True
    free = (~used).nonzero()[:, 0]
    need = (length + extra + P - 1) // P - full - keep.long()
    offset = need.cumsum(0) - need
    base = full + keep.long()
    fresh = free[(offset[:, None] + col - base[:, None]).clamp(0, len(free) - 1)]
    out = torch.where(col < base[:, None], t, torch.where(col < (base + need)[:, None], fresh, -1)).int()
    copy = part & ~keep
    src, dst = last[copy], free[offset[copy]]
    for name in ("k_codes", "v_codes", "k_scale", "v_scale"):
        s[name][:, dst] = s[name][:, src]
    return [out, (length + extra).int()]


def _plain_compact(s):
    case, tables, P, N = s["case"], s["tables"], s["case"]["page"], s["case"]["pages"]
    live = torch.arange(tables.shape[1], device="cuda") < ((s["lengths"] + P - 1) // P)[:, None]
    used = torch.zeros(N, dtype=torch.bool, device="cuda")
    used[tables[live].long()] = True
    ids = torch.arange(N, device="cuda")
    count = used.sum()
    src, dst = ids[used & (ids >= count)], ids[~used & (ids < count)]
    to = ids.clone()
    to[src] = dst
    for name in ("k_codes", "v_codes", "k_scale", "v_scale"):
        s[name][:, dst] = s[name][:, src]
    return [torch.where(live, to[tables.clamp(min=0).long()], -1).int()]


def _pools(s):
    # pages are moved as they are, byte for byte: the pool's codes and scales themselves
    return [s[name] for name in ("k_codes", "k_scale", "v_codes", "v_scale")]


def run(s):
    case = s["case"]
    op = case["op"]
    if not own:
        if op == "rotary":
            x = s["x"]
            return _rotate(x.float(), s["cos_sin"][s["positions"].long()], case["interleaved"], case["inverse"]).to(x.dtype)
        if op == "append":
            return _plain_append(s)
        if op == "attend":
            return _plain_attend(s)
        return (_plain_fork(s) if op == "fork" else _plain_compact(s)) + _pools(s)
    if op == "rotary":
        from ffn_residual_mesh_b200.kvcache import rotary
        return rotary(s["x"], s["positions"], s["rope"], inverse=case["inverse"])
    cache = s["cache"]
    if op == "append":
        starts = None if case["chunk"] == 1 else s["starts"]
        q = cache.append(0, s["k"], s["v"], s["tables"], s["lengths"], starts=starts, rope=s["rope"], q=s["q"])
        return [q, *cache.read(0, s["tables"], s["lengths"], s["seen"], s["rows"], dtype=torch.float32)]
    if op == "attend":
        return cache.attend(0, s["q"], s["tables"], s["lengths"], starts=s["starts"], window=case["window"])
    if op == "fork":
        tables, lengths, _ = cache.fork(s["tables"], s["lengths"], s["parents"], s["extra"])
        return [tables, lengths] + _pools(s)
    tables, _ = cache.compact(s["tables"], s["lengths"])
    return [tables] + _pools(s)


# ------------------------------------------------------------------------------- the same in 64 bits
def _turn64(x, cos_sin, pos, interleaved, sign=1.0):
    R = cos_sin.shape[1]
    z = x.double().clone()
    ang = torch.complex(cos_sin[pos, :R // 2].double(), sign * cos_sin[pos, R // 2:].double())[:, None]
    if interleaved:
        pair = torch.view_as_complex(z[..., :R].reshape(*z.shape[:-1], R // 2, 2).contiguous()) * ang
        z[..., :R] = torch.view_as_real(pair).reshape(*z.shape[:-1], R)
    else:
        pair = torch.complex(z[..., :R // 2], z[..., R // 2:R]) * ang
        z[..., :R // 2], z[..., R // 2:R] = pair.real, pair.imag
    return z


def exact(case, seed):
    global own
    was, own = own, False
    s = prepare(case, seed)
    own = was
    op = case["op"]
    if op == "rotary":
        return _turn64(s["x"], s["cos_sin"], s["positions"].long(), case["interleaved"], -1.0 if case["inverse"] else 1.0)
    if op == "append":
        return _exact_append(case, s)
    if op == "attend":
        return _exact_attend(case, s)
    return None  # page numbers and moved bytes: whole values


def _exact_append(case, s):
    P, (new, lengths) = case["page"], _append_shape(case)
    table, at = s["tables"].tolist(), _rows(new)
    pos = torch.cat([torch.arange(a - n, a) for n, a in zip(new, lengths)]).cuda()
    out = [_turn64(s["q"], s["cos_sin"], pos, case["interleaved"])]
    k = _turn64(s["k"], s["cos_sin"], pos, case["interleaved"])
    for x, codes, scale in ((k, s["k_codes"][0], s["k_scale"][0]), (s["v"].double(), s["v_codes"][0], s["v_scale"][0])):
        got = []
        for b, (n, a) in enumerate(zip(new, lengths)):
            for first in range((a - n) // P * P, a, P):
                page, held = table[b][first // P], max(0, a - n - first)
                lo, hi = max(first, a - n), min(first + P, a)
                rows = x[at[b] + lo - (a - n):at[b] + hi - (a - n)]  # [new, heads, D]
                before = scale[page].double() if held else torch.zeros_like(scale[page], dtype=torch.float64)
                step = torch.maximum(before, rows.abs().amax((0, 2)) / 127).clamp(min=1e-12)
                old = (codes[page, :, :held].double() * (before / step)[:, None, None]).round().transpose(0, 1)
                fresh = (rows / step[:, None]).round().clamp(-127, 127)
                got.append(torch.cat([old, fresh]) * step[:, None])
        out.append(torch.cat(got))
    return out


def _exact_attend(case, s):
    P, G, D, Hk = case["page"], case["group"], case["dim"], case["kv_heads"]
    new, lengths = _attend_shape(case)
    at = _rows(new)
    out = torch.zeros(at[-1], Hk, G, D, dtype=torch.float64, device="cuda")
    for b, (n, a) in enumerate(zip(new, lengths)):
        if a == 0:
            continue
        pages = s["tables"][b, :-(-a // P)].long()
        key, pos = torch.arange(a, device="cuda"), torch.arange(a - n, a, device="cuda")
        for h in range(Hk):
            k, v = [(s[c][0][pages, h].double() * s[f][0][pages, h].double()[:, None, None]).reshape(-1, D)[:a]
                    for c, f in (("k_codes", "k_scale"), ("v_codes", "v_scale"))]
            for lo in range(0, n, 1024):
                p = pos[lo:lo + 1024]
                hidden = key > p[:, None]
                if case["window"]:
                    hidden |= key <= p[:, None] - case["window"]
                q = s["q"][at[b] + lo:at[b] + lo + len(p)].view(len(p), Hk, G, D)[:, h].double()
                y = torch.einsum("tgd,kd->gtk", q, k) / math.sqrt(D)
                y = torch.softmax(y.masked_fill_(hidden, float("-inf")), -1)
                out[at[b] + lo:at[b] + lo + len(p), h] = torch.einsum("gtk,kd->tgd", y, v)
    return out.view(at[-1], Hk * G, D)
