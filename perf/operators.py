"""The paged 8-bit key/value cache and the attention over it, as cases that a timing program can run.

Three operators: `append` writes the keys and values of new tokens into the cache (int8 codes with one 32-bit scale
for each block of 32 tokens and head), `attend` is attention of query rows over the cache, and `pages` is the
bookkeeping of the cache's pages on the GPU (fork, free, compact, reserve), which copies pages.

The cache is the caller's memory:

  codes  int8  [layers][pages][K, V][heads][blocks of 32 tokens][32 * D]
           K block: [D / 16][32 tokens][16]: byte (c, t, i) is dimension 16 c + i of token t
           V block: [2][D][16]: byte (h, d, 8 (a & 1) + 4 (a >> 1) + b) is dimension d of token 8 a + 4 h + b (a, b < 4)
  scales f32   [layers][pages][K, V][heads][blocks]
  table  int32 [slots][most pages]   the pages of each sequence
  len    int32 [slots]               its tokens
  ref    int32 [pages]               how many sequences hold a page (0: free)

Where `own` is false, the operators run in elementary torch operations on the same memory.
"""
import math
import random

import torch

own = False

BLOCK = 32  # tokens of a scale
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _attend(name, seqs, len_min, len_max, rows_min, rows_max, heads, kv_heads, dim, page, dtype, softcap=0.0, window=0,
            alibi=False, causal=True, len_seed=1):
    return {"name": name, "op": "attend", "seqs": seqs, "len_min": len_min, "len_max": len_max, "rows_min": rows_min,
            "rows_max": rows_max, "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page, "dtype": dtype,
            "softcap": softcap, "window": window, "alibi": alibi, "causal": causal, "len_seed": len_seed}


def _append(name, seqs, len_min, len_max, rows_min, rows_max, kv_heads, dim, page, dtype, len_seed=1):
    return {"name": name, "op": "append", "seqs": seqs, "len_min": len_min, "len_max": len_max, "rows_min": rows_min,
            "rows_max": rows_max, "kv_heads": kv_heads, "dim": dim, "page": page, "dtype": dtype, "len_seed": len_seed}


def _pages(name, kind, seqs, children, len_min, len_max, layers, kv_heads, dim, page, len_seed=1):
    return {"name": name, "op": "pages", "kind": kind, "seqs": seqs, "children": children, "len_min": len_min,
            "len_max": len_max, "layers": layers, "kv_heads": kv_heads, "dim": dim, "page": page, "len_seed": len_seed}


def listed():
    return [
        # generating text for one user, a short conversation: nothing but latency
        _attend("attend-one", 1, 301, 301, 1, 1, 32, 8, 128, 32, "f32"),
        # one user with a very long document in the cache
        _attend("attend-long", 1, 131009, 131009, 1, 1, 32, 8, 128, 64, "bf16"),
        # a serving batch, conversations of very different lengths
        _attend("attend-batch", 64, 150, 8000, 1, 1, 32, 8, 128, 64, "bf16", len_seed=3),
        # the same without shared heads, an odd batch and head size
        _attend("attend-heads", 17, 40, 3000, 1, 1, 16, 16, 96, 32, "f16", len_seed=5),
        # draft tokens to verify, wide heads with capped scores and a sliding window
        _attend("attend-draft", 8, 900, 4000, 5, 5, 16, 8, 256, 32, "f32", softcap=50.0, window=1024, len_seed=7),
        # a prompt of one user, and pieces of several prompts behind what is cached of them, with distance biases
        _attend("attend-prompt", 1, 6011, 6011, 6011, 6011, 32, 8, 128, 64, "bf16"),
        _attend("attend-pieces", 5, 100, 5000, 1, 700, 16, 4, 64, 128, "f32", alibi=True, len_seed=11),
        # a step of a serving batch, a prompt, and pieces that begin and end inside a block
        _append("append-step", 64, 1, 60, 1, 1, 8, 128, 64, "f32", len_seed=13),
        _append("append-prompt", 1, 8191, 8191, 8191, 8191, 8, 128, 64, "bf16"),
        _append("append-pieces", 9, 30, 1500, 1, 700, 5, 96, 32, "f16", len_seed=17),
        # several answers to each prompt: the full pages are shared, the last one is copied
        _pages("pages-fork", "fork", 2, 4, 300, 900, 4, 8, 128, 64, len_seed=19),
        # half of a batch ends: its pages are freed, the others move together, new sequences take what is free
        _pages("pages-compact", "compact", 64, 0, 400, 2000, 8, 8, 128, 64, len_seed=23),
    ]


def draw(rng):
    def spread(lo, hi):
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))

    op = rng.choice(["attend"] * 6 + ["append"] * 2 + ["pages"] * 2)
    dim, page = 32 * rng.choice([2, 3, 4, 4, 4, 6, 8]), rng.choice([32, 64, 128])
    kv_heads = rng.choice([1, 2, 3, 4, 5, 8, 8, 16])
    dtype, seed = rng.choice(["f32", "f16", "bf16"]), rng.randint(1, 10 ** 6)
    if op == "attend":
        heads = kv_heads * rng.choice([1, 2, 3, 4, 5, 8])
        kind = rng.choice(["step", "step", "draft", "pieces"])
        seqs = spread(1, 96) if kind == "step" else spread(1, 12)
        longest = spread(1, max(64, 262144 // seqs))
        rows = {"step": (1, 1), "draft": (2, 8)}.get(kind) or (1, min(longest, spread(16, 3000)))
        case = _attend("", seqs, max(1, longest // rng.choice([1, 3, 30])), longest, rows[0], max(rows), heads, kv_heads,
                       dim, page, dtype, softcap=rng.choice([0.0, 0.0, 30.0]), window=rng.choice([0, 0, spread(1, 4096)]),
                       alibi=rng.random() < 0.2, causal=rng.random() < 0.9, len_seed=seed)
        while (work(case)["bytes"] > 2.7e8 or work(case)["flops"] > 2.9e11 or 2 * seqs * case["len_max"] * kv_heads * dim > 6e8
               or seqs * heads * case["rows_max"] * case["len_max"] > 1.2e9):
            case["len_max"] = max(1, case["len_max"] // 2)
            case["len_min"] = min(case["len_min"], case["len_max"])
            case["rows_max"] = max(case["rows_min"], min(case["rows_max"], case["len_max"]))
    elif op == "append":
        seqs, rows = spread(1, 96), rng.choice([1, 1, 5, spread(8, 4000)])
        case = _append("", seqs, max(1, rows // 2), rows + rng.randint(0, 200), 1, rows, kv_heads, dim, page, dtype, len_seed=seed)
        while case["seqs"] * case["len_max"] > 16000:
            case["seqs"] = max(1, case["seqs"] // 2)
    else:
        case = _pages("", rng.choice(["fork", "compact"]), spread(2, 48), rng.randint(1, 6), 1, spread(64, 1500), rng.randint(1, 6),
                      kv_heads, dim, page, len_seed=seed)
        while work(case)["bytes"] > 9e8 and case["layers"] > 1:
            case["layers"] -= 1
        while work(case)["bytes"] > 9e8:
            case["seqs"] //= 2
    del case["name"]
    return case


def _lengths(case):
    """(tokens in the cache, rows of this call) of each sequence; the rows are the last of the tokens."""
    r = random.Random(case["len_seed"])
    got = []
    for _ in range(case["seqs"]):
        length = int(round(math.exp(r.uniform(math.log(case["len_min"]), math.log(case["len_max"])))))
        rows = r.randint(case["rows_min"], case["rows_max"]) if "rows_min" in case else 0
        got.append((max(length, rows), rows))
    return got


# ------------------------------------------------------------------------------------------ inputs


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed * 7919 + 17)
    cpu = random.Random(seed)
    op, D, H, P = case["op"], case["dim"], case["kv_heads"], case["page"]
    B, layers = case["seqs"], case.get("layers", 1)
    lengths = _lengths(case)
    held = [-(-length // P) for length, _ in lengths]
    slots = B * (1 + case.get("children", 0))
    most = max(held) + 1
    n_pages = sum(held) + max(4, sum(held) // 8) + 3 * (slots - B)
    order = list(range(n_pages))  # where the pages lie after some hours of use
    cpu.shuffle(order)
    table, at = [[0] * most for _ in range(slots)], 0
    for i, n in enumerate(held):
        table[i][:n] = order[at:at + n]
        at += n
    ref = [0] * n_pages
    for p in order[:at]:
        ref[p] = 1

    codes = torch.empty(layers, n_pages, 2, H, P // BLOCK, BLOCK * D, dtype=torch.int8, device="cuda")
    for layer in range(layers):
        codes[layer] = (torch.randn(codes.shape[1:], device="cuda", generator=g) * 40).round().clamp(-127, 127).to(torch.int8)
    scales = 0.02 + 0.01 * torch.rand(codes.shape[:-1], device="cuda", generator=g)
    s = {"case": dict(case), "codes": codes, "scales": scales, "table": _ints(table), "ref": _ints(ref),
         "len": _ints([length for length, _ in lengths] + [0] * (slots - B))}
    if op == "pages":
        if case["kind"] == "fork":
            s["src"] = _ints([i for i in range(B) for _ in range(case["children"])])
            s["dst"] = _ints(list(range(B, slots)))
        else:  # two halves of the batch, which end in turn
            s["turn"] = 0
            s["half"] = [_ints(list(range(k, B, 2))) for k in (0, 1)]
            s["new"] = [s["len"][h.long()].clone() for h in s["half"]]
    else:
        rows = [n for _, n in lengths]
        s["row_start"] = _ints([sum(rows[:i]) for i in range(B + 1)])
        s["n_rows"], s["max_rows"], s["max_len"] = sum(rows), max(rows), max(length for length, _ in lengths)
        dt = DTYPES[case["dtype"]]
        if op == "append":  # a few channels of the keys are larger than the others
            channel = 1 + 3 * (torch.rand(H, D, device="cuda", generator=g) > 0.95)
            s["k"] = (torch.randn(s["n_rows"], H, D, device="cuda", generator=g) * channel).to(dt)
            s["v"] = torch.randn(s["n_rows"], H, D, device="cuda", generator=g).to(dt)
        else:  # some heads look closer than others
            sharp = 0.5 + 2 * torch.rand(case["heads"], 1, device="cuda", generator=g)
            s["q"] = (torch.randn(s["n_rows"], case["heads"], D, device="cuda", generator=g) * sharp).to(dt)
            s["out"] = torch.empty_like(s["q"])
            n = case["heads"]
            s["alibi"] = 2.0 ** (-8.0 * torch.arange(1, n + 1, device="cuda") / n) if case["alibi"] else None
    if own:  # the handles that a program keeps
        _handles(s)
    return s


def _handles(s):
    from jxai_amd import formats, kv

    c, codes = s["case"], s["codes"]
    s["cache"] = kv.KVCache(n_layers=codes.shape[0], n_pages=codes.shape[1], page_tokens=c["page"], n_kv_heads=c["kv_heads"],
                            head_dim=c["dim"], max_seqs=s["table"].shape[0], max_pages=s["table"].shape[1],
                            buffers={name: s[name] for name in ("codes", "scales", "table", "len", "ref")})
    if c["op"] == "pages":
        return
    s["type"] = {"f32": formats.F32, "f16": formats.F16, "bf16": formats.BF16}[c["dtype"]]
    s["batch"] = kv.KVBatch(n_seqs=c["seqs"], n_rows=s["n_rows"], max_rows=s["max_rows"], max_len=s["max_len"],
                            row_start=s["row_start"])
    if c["op"] == "attend":
        s["attention"] = kv.Attention(n_heads=c["heads"], dtype=s["type"], scale=c["dim"] ** -0.5, softcap=c["softcap"],
                                      window=c["window"], causal=c["causal"], alibi=s["alibi"])
        s["ws"] = s["cache"].workspace(s["batch"], s["attention"])


# ------------------------------------------------------------------------------------------ one pass


def run(s):
    c = s["case"]
    if c["op"] == "attend":
        if own:
            s["cache"].attend(s["batch"], s["attention"], s["q"], s["out"], s["ws"])
            return s["out"]
        return _plain_attend(s)
    if c["op"] == "append":
        if own:
            s["cache"].append(s["batch"], s["k"], s["v"], s["type"])
        else:
            _plain_append(s)
        # the 8-bit values as what they stand for
        return {"values": s["codes"] * s["scales"][..., None], "scales": s["scales"]}
    if c["kind"] == "fork":
        if own:
            s["cache"].fork(s["src"], s["dst"], s["src"].numel())
        else:
            _plain_fork(s)
    else:
        half, new = s["half"][s["turn"]], s["new"][s["turn"]]
        s["turn"] ^= 1
        if own:
            s["cache"].trim(half, None, half.numel())
            s["cache"].compact()
            s["cache"].reserve(half, new, half.numel())
        else:
            _plain_free(s, half)
            _plain_compact(s)
            _plain_reserve(s, half, new)
    # pages are moved as bytes, whatever they hold
    return {name: s[name] for name in ("table", "len", "ref", "codes", "scales")}


# ------------------------------------------------------------------------------------------ plain forms


def _gathered(s, layer=0):
    """Keys and values of every sequence in 32 bits, [sequences][kv heads][tokens up to the longest][D]."""
    c = s["case"]
    D, H, n = c["dim"], c["kv_heads"], -(-s["max_len"] // c["page"])
    pages = s["table"][:, :n].long()
    codes, scales = s["codes"][layer][pages], s["scales"][layer][pages]  # [B][n][2][H][blocks][...]
    B, blocks = pages.shape[0], codes.shape[4]
    x = codes.float() * scales[..., None]
    k = x[:, :, 0].reshape(B, n, H, blocks, D // 16, BLOCK, 16).permute(0, 2, 1, 3, 5, 4, 6).reshape(B, H, -1, D)
    # [h][d][a & 1][a >> 1][b] -> [a >> 1][a & 1][h][b][d]
    v = x[:, :, 1].reshape(B, n, H, blocks, 2, D, 2, 2, 4).permute(0, 2, 1, 3, 7, 6, 4, 8, 5).reshape(B, H, -1, D)
    return k, v


def _rows(s):
    """(sequence, place in it) of each row."""
    at = torch.arange(s["n_rows"], device="cuda")
    seq = (at[:, None] >= s["row_start"][None, 1:]).sum(1)
    return seq, at - s["row_start"].long()[seq]


def _plain_attend(s):
    c = s["case"]
    H, D, n = c["kv_heads"], c["dim"], s["max_rows"]
    G = c["heads"] // H
    k, v = _gathered(s)
    B, T = k.shape[0], k.shape[2]
    seq, place = _rows(s)
    q = torch.zeros(B, n, H, G, D, device="cuda")
    q[seq, place] = s["q"].float().reshape(-1, H, G, D)
    q = q.permute(0, 2, 3, 1, 4).reshape(B, H, G * n, D)
    x = torch.matmul(q, k.transpose(2, 3).contiguous()) * D ** -0.5
    del k
    if c["softcap"]:
        x = c["softcap"] * torch.tanh(x / c["softcap"])
    x = x.reshape(B, H, G, n, T)
    rows = s["row_start"][1:] - s["row_start"][:-1]
    pos = (s["len"] - rows)[:, None] + torch.arange(n, device="cuda")  # [B][n]
    t = torch.arange(T, device="cuda")
    if s["alibi"] is not None:
        x = x + s["alibi"].reshape(1, H, G, 1, 1) * (t - pos[:, :, None]).float()[:, None, None]
    seen = (t < s["len"][:, None, None]).expand(B, n, T)
    if c["causal"]:
        seen = seen & (t <= pos[:, :, None])
    if c["window"]:
        seen = seen & (t > pos[:, :, None] - c["window"])
    x = x.masked_fill(~seen[:, None, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(top == -math.inf, torch.zeros_like(top), top))
    del x
    total = p.sum(-1, keepdim=True)
    y = torch.matmul(p.reshape(B, H, G * n, T), v).reshape(B, H, G, n, D) / torch.where(total == 0, torch.ones_like(total), total)
    return y.permute(0, 3, 1, 2, 4)[seq, place].reshape(s["n_rows"], c["heads"], D).to(s["q"].dtype)


def _plain_append(s, layer=0):
    c = s["case"]
    H, D, P = c["kv_heads"], c["dim"], c["page"]
    rows = s["row_start"][1:] - s["row_start"][:-1]
    begin = (s["len"] - rows).long()
    block = begin[:, None] // BLOCK + torch.arange((s["max_rows"] + BLOCK - 2) // BLOCK + 1, device="cuda")
    sequence, nth = (block * BLOCK < s["len"][:, None]).nonzero(as_tuple=True)  # every block that gets a token
    block = block[sequence, nth]
    token = block[:, None] * BLOCK + torch.arange(BLOCK, device="cuda")  # [N][32]
    first = begin[sequence][:, None]
    new, old = (token >= first) & (token < s["len"][sequence][:, None]), token < first
    row = (s["row_start"][sequence].long()[:, None] + token - first).clamp(0, s["n_rows"] - 1)
    page, inside = s["table"][sequence, block * BLOCK // P].long(), block % (P // BLOCK)
    for which, x in ((0, s["k"]), (1, s["v"])):
        x = x[row].float() * new[:, :, None, None]  # [N][32][H][D]
        before = s["scales"][layer, page, which, :, inside] * old.any(1)[:, None]  # [N][H]
        top = (x.abs().amax((1, 3)).double() / 127).float()
        top = torch.where(top < 2.0 ** -120, torch.zeros_like(top), top)
        now = torch.maximum(before, top)
        step = torch.where(now > 0, now, torch.ones_like(now)).double()[:, None, :, None]
        # the nearest code: the quotient in 64 bits, or values next to the middle of two codes would go astray
        q = torch.where(now[:, None, :, None] > 0, (x.double() / step).round(), torch.zeros_like(step)).clamp(-127, 127)
        shape = (-1, H, D // 16, BLOCK, 16) if which == 0 else (-1, H, 2, D, 2, 2, 4)
        to, back = ((0, 3, 1, 2, 4), (0, 2, 3, 1, 4)) if which == 0 else ((0, 5, 4, 2, 6, 1, 3), None)
        held = s["codes"][layer, page, which, :, inside].reshape(shape).permute(to).reshape(-1, BLOCK, H, D)
        kept = torch.where(old[:, :, None, None], (held.double() * before.double()[:, None, :, None] / step).round(), held.double())
        q = torch.where(new[:, :, None, None], q, kept).to(torch.int8)
        if which == 0:
            q = q.reshape(-1, BLOCK, H, D // 16, 16).permute(back)
        else:
            q = q.reshape(-1, 2, 2, 2, 4, H, D).permute(0, 5, 3, 6, 2, 1, 4)
        s["codes"][layer, page, which, :, inside] = q.reshape(-1, H, BLOCK * D)
        s["scales"][layer, page, which, :, inside] = now


def _pages_of(s, length):
    return (length + s["case"]["page"] - 1) // s["case"]["page"]


def _places(s):
    return torch.arange(s["table"].shape[1], device="cuda")


def _count(s, table, mask, by):
    s["ref"].index_add_(0, table.reshape(-1), mask.reshape(-1).int() * by)


def _plain_fork(s):
    P, src, dst = s["case"]["page"], s["src"].long(), s["dst"].long()
    length, parent, former = s["len"][src], s["table"][src], s["table"][dst]
    free = torch.argsort(s["ref"] > 0, stable=True)
    partial = (length % P > 0).int()
    fresh = free[partial.cumsum(0) - partial].int()
    full = (length // P)[:, None]
    at = _places(s)
    _count(s, parent, at < full, 1)
    _count(s, former, at < _pages_of(s, s["len"][dst])[:, None], -1)
    _count(s, fresh, partial, 1)
    last = (at == full) & (partial[:, None] > 0)
    s["table"][dst] = torch.where(at < full, parent, torch.where(last, fresh[:, None], former))
    s["len"][dst] = length
    tail = torch.gather(parent, 1, full.long().clamp(max=parent.shape[1] - 1))[:, 0]
    to, of = fresh[partial > 0].long(), tail[partial > 0].long()
    for name in ("codes", "scales"):
        s[name][:, to] = s[name][:, of]


def _plain_free(s, slots):
    slots = slots.long()
    _count(s, s["table"][slots], _places(s) < _pages_of(s, s["len"][slots])[:, None], -1)
    s["len"][slots] = 0


def _plain_compact(s):
    live, at = s["ref"] > 0, torch.arange(s["ref"].numel(), device="cuda")
    count = live.sum()
    of, to = (live & (at >= count)).nonzero()[:, 0], (~live & (at < count)).nonzero()[:, 0]
    moved = at.int()
    moved[of] = to.int()
    for name in ("codes", "scales"):
        s[name][:, to] = s[name][:, of]
    s["ref"][to] = s["ref"][of]
    s["ref"][of] = 0
    s["table"].copy_(torch.where(_places(s) < _pages_of(s, s["len"])[:, None], moved[s["table"].long()], s["table"]))


def _plain_reserve(s, slots, new):
    slots = slots.long()
    held, needed = _pages_of(s, s["len"][slots]), _pages_of(s, s["len"][slots] + new)
    begin = (needed - held).cumsum(0) - (needed - held)
    free = torch.argsort(s["ref"] > 0, stable=True)
    at = _places(s)
    take = (at >= held[:, None]) & (at < needed[:, None])
    fresh = free[(begin[:, None] + at - held[:, None]).clamp(0, free.numel() - 1)].int()
    s["table"][slots] = torch.where(take, fresh, s["table"][slots])
    _count(s, fresh, take, 1)
    s["len"][slots] += new


# ------------------------------------------------------------------------------------------ what a pass needs


def work(case):
    D, H, P = case["dim"], case["kv_heads"], case["page"]
    lengths = _lengths(case)
    block = 2 * H * (BLOCK * D + 4)  # codes and scales of 32 tokens in one layer
    if case["op"] == "pages":
        page = case["layers"] * block * P // BLOCK
        if case["kind"] == "fork":
            moved = case["children"] * sum(length % P > 0 for length, _ in lengths)
        else:
            held = [-(-length // P) for length, _ in lengths]
            moved = min(sum(held[0::2]), sum(held[1::2]))
        return {"bytes": 2 * moved * page + 4 * sum(length // P + 1 for length, _ in lengths), "flops": 0}
    size = {"f32": 4, "f16": 2, "bf16": 2}[case["dtype"]]
    if case["op"] == "append":  # the values in, their codes out, and the cache's values as they are returned
        pages = sum(-(-length // P) for length, _ in lengths)
        return {"bytes": sum(n for _, n in lengths) * 2 * H * D * (size + 1) + pages * 2 * H * P * D * 5, "flops": 0}
    tokens, pairs = 0, 0
    for length, n in lengths:
        begin = length - n
        last = [min(length, begin + i + 1) if case["causal"] else length for i in range(n)]
        first = [max(0, begin + i + 1 - case["window"]) if case["window"] else 0 for i in range(n)]
        tokens += max(0, max(last) - min(first))
        pairs += sum(max(0, b - a) for a, b in zip(first, last))
    rows = sum(n for _, n in lengths)
    return {"bytes": tokens * block / BLOCK + 2 * rows * case["heads"] * D * size, "flops": 4 * pairs * case["heads"] * D}


# ------------------------------------------------------------------------------------------ in 64 bits


def _tokens64(s, slot, which, head, length):
    """Tokens 0 .. length of one sequence and head in 64 bits, from the layout's definition."""
    P, D = s["case"]["page"], s["case"]["dim"]
    t = torch.arange(length, device="cuda")
    page, inside, r = s["table"][slot].long()[t // P], t % P // BLOCK, t % BLOCK
    d = torch.arange(D, device="cuda")
    if which == 0:
        byte = (d // 16 * BLOCK)[None] * 16 + r[:, None] * 16 + d % 16
    else:
        a, h, b = r // 8, r // 4 % 2, r % 4
        byte = (h[:, None] * D + d) * 16 + (8 * (a % 2) + 4 * (a // 2) + b)[:, None]
    flat = s["codes"][0, :, which, head]
    return flat[page[:, None], inside[:, None], byte].double() * s["scales"][0, page, which, head, inside].double()[:, None]


def exact(case, seed):
    if case["op"] == "pages":
        return None
    s = prepare(case, seed)
    lengths = _lengths(case)
    if case["op"] == "append":
        values = s["codes"].double() * s["scales"].double()[..., None]
        scales = s["scales"].double()
        D, P = case["dim"], case["page"]
        d = torch.arange(D, device="cuda")
        row = 0
        for i, (length, n) in enumerate(lengths):
            for begin in range((length - n) // BLOCK * BLOCK, length, BLOCK):
                page, inside = int(s["table"][i, begin // P]), begin % P // BLOCK
                lo, hi = max(begin, length - n), min(begin + BLOCK, length)
                r = torch.arange(BLOCK, device="cuda")
                kbyte = (d // 16 * BLOCK)[None] * 16 + r[:, None] * 16 + d % 16
                a, h, b = r // 8, r // 4 % 2, r % 4
                vbyte = (h[:, None] * D + d) * 16 + (8 * (a % 2) + 4 * (a // 2) + b)[:, None]
                for which, x, byte in ((0, s["k"], kbyte), (1, s["v"], vbyte)):
                    x = x[row + lo - (length - n):row + hi - (length - n)].double()  # [m][H][D]
                    before = scales[0, page, which, :, inside].clone() if lo > begin else torch.zeros(x.shape[1], device="cuda").double()
                    now = torch.maximum(before, (x.abs().amax((0, 2)) / 127.0).float().double())  # held in 32 bits
                    cells = values[0, page, which, :, inside]  # [H][32 * D], a view
                    if lo > begin:
                        kept = cells[:, byte[:lo - begin].reshape(-1)]
                        cells[:, byte[:lo - begin].reshape(-1)] = (kept / now[:, None]).round() * now[:, None]
                    q = (x / now[None, :, None]).round() * now[None, :, None]
                    cells[:, byte[lo - begin:hi - begin].reshape(-1)] = q.permute(1, 0, 2).reshape(q.shape[1], -1)
                    if hi < begin + BLOCK:  # codes behind the last token keep their bytes
                        rest = byte[hi - begin:].reshape(-1)
                        cells[:, rest] = s["codes"][0, page, which, :, inside][:, rest].double() * now[:, None]
                    scales[0, page, which, :, inside] = now
            row += n
        return {"values": values, "scales": scales}
    if sum(length for length, _ in lengths) * case["heads"] > 3e7:
        return None
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    G, row = case["heads"] // case["kv_heads"], 0
    for i, (length, n) in enumerate(lengths):
        t, p = torch.arange(length, device="cuda"), torch.arange(length - n, length, device="cuda")
        hidden = torch.zeros(n, length, dtype=torch.bool, device="cuda")
        if case["causal"]:
            hidden |= t[None] > p[:, None]
        if case["window"]:
            hidden |= t[None] <= p[:, None] - case["window"]
        for kv_head in range(case["kv_heads"]):
            k, v = _tokens64(s, i, 0, kv_head, length), _tokens64(s, i, 1, kv_head, length)
            for head in range(kv_head * G, kv_head * G + G):
                x = s["q"][row:row + n, head].double() @ k.T.contiguous() / math.sqrt(case["dim"])
                if case["softcap"]:
                    x = (x / case["softcap"]).tanh() * case["softcap"]
                if s["alibi"] is not None:
                    x = x - (p[:, None] - t[None]) * s["alibi"][head].double()
                x = x.masked_fill(hidden, -math.inf)
                out[row:row + n, head] = torch.nan_to_num(torch.softmax(x, 1)) @ v
        row += n
    return out
