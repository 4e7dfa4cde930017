"""Timed cases of the paged K/V cache: many sequences on one pool of pages.

Four operators, each in its plain form (elementary torch operations in 32 bits, angles in 64) and, with `own` set, as a
program calls the library (mechta_amd.paged):

- `attend`: a batch of sequences, each with a chunk of new tokens (one for generation, a few for the verify of drafted
  tokens, hundreds for a prompt), attends causally over its pages: grouped query heads, optionally a sliding window,
  a sink logit per head, and the sigmoid gate on the output.
- `append`: the batch's new K rows rotated at their positions and written with V into the pages, q rotated beside.
- `rotate`: rotary positions alone, on rows at given positions: pairs half a rotated part apart or neighbours, part of
  the head, scaled for long contexts.
- `fork` / `compact`: copies of pages over all layers: samples forked off one prompt, and a pool whose holes are closed.

Ranges: 1 to 64 sequences, 1 to 131,072 positions, 1 to 4,096 tokens a batch (8,192 for append and rotate), head
sizes 64, 128 and 256, 1 to 16 query heads per K/V head, pages of 32 to 256 positions, f16 and bf16 (f32 too for
rotate). The cache is written in turns over the sequences, as it is when they grow side by side, so a sequence's pages
lie scattered.
"""
import math

import torch

own = False

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
TURNS = 8  # turns in which the sequences of a cache were written


def listed():
    return [
        # the first answer after a greeting: one token, a handful of positions: the latency of a call
        dict(name="attend_1tok_17", op="attend", type="f16", q_heads=16, kv_heads=2, dim=256, page=64, counts="1",
             lens="17", window=0, sinks=False, gate=True),
        # 64 conversations generating side by side, lengths from a question to a document
        dict(name="attend_64seq_decode", op="attend", type="bf16", q_heads=32, kv_heads=4, dim=128, page=64,
             counts="1x64", lens="log 500 8001", window=0, sinks=False, gate=False),
        # the verify of three drafted tokens in a long conversation
        dict(name="attend_verify4_64k", op="attend", type="f16", q_heads=16, kv_heads=2, dim=256, page=128, counts="4",
             lens="65540", window=0, sinks=False, gate=True),
        # a 512-token chunk of a long prompt
        dict(name="attend_chunk512_9k", op="attend", type="f16", q_heads=16, kv_heads=2, dim=256, page=64, counts="512",
             lens="9512", window=0, sinks=False, gate=True),
        # a sliding layer of a batch in which prompts arrive while others generate, with sinks, on small pages
        dict(name="attend_mixed_window", op="attend", type="bf16", q_heads=32, kv_heads=4, dim=128, page=32,
             counts="700 256 33 1x12", lens="700 3001 97 1200 64 513 514 3999 2048 5 777 900 1500 4001 1", window=513,
             sinks=True, gate=False),
        # a whole prompt at once, the matrix units' case
        dict(name="attend_prompt_4k", op="attend", type="bf16", q_heads=32, kv_heads=4, dim=128, page=64, counts="4096",
             lens="4096", window=0, sinks=False, gate=False),
        # one step of 64 generating conversations: a token each, a quarter of the head rotated
        dict(name="append_64seq", op="append", type="f16", q_heads=16, kv_heads=2, dim=256, page=64, counts="1x64",
             lens="log 100 4000", rot=64, layout="half", scaling="none", base=1e7, factor=1.0, original=0),
        # the prompts of four conversations, ragged, the whole head rotated, positions scaled
        dict(name="append_4prompts", op="append", type="bf16", q_heads=32, kv_heads=4, dim=128, page=64,
             counts="4096 2500 1031 565", lens="4096 2777 9000 565", rot=128, layout="interleaved", scaling="bands",
             base=5e5, factor=8.0, original=8192),
        # the query heads of one token, in 32 bits
        dict(name="rotate_1tok", op="rotate", type="f32", rows=1, heads=16, dim=256, rot=64, layout="half",
             scaling="none", base=1e7, factor=1.0, original=0, positions=65536),
        # a prompt's query heads, context stretched 32 times
        dict(name="rotate_8k", op="rotate", type="bf16", rows=8192, heads=32, dim=128, rot=128, layout="half",
             scaling="yarn", base=1e4, factor=32.0, original=4096, positions=131072),
        # eight samples off one prompt: the partly filled last page copied for each, all layers
        dict(name="fork_8", op="fork", type="f16", layers=10, kv_heads=2, dim=256, page=64, length=5000, children=8),
        # a conversation moved down over freed pages and copied for a second reader, all layers
        dict(name="compact_16k", op="compact", type="f16", layers=10, kv_heads=2, dim=256, page=64, pages=256),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "append", "rotate", "fork", "compact"])
    kv, group, dim = rng.choice([1, 2, 3, 4, 8]), rng.choice([1, 2, 4, 5, 8, 16]), rng.choice([64, 128, 256])
    c = dict(op=op, type=rng.choice(["f16", "bf16"]), kv_heads=kv, dim=dim, page=rng.choice([32, 64, 128, 256]))
    rope = dict(rot=rng.choice([dim, dim // 2, dim // 4]), layout=rng.choice(["half", "interleaved"]),
                scaling=rng.choice(["none", "linear", "ntk", "yarn", "bands"]), base=rng.choice([1e4, 5e5, 1e7]),
                factor=rng.choice([2.0, 8.0, 32.0]), original=rng.choice([4096, 8192]))
    if op == "rotate":
        rows = _log(rng, 1, 8192)
        heads = rng.choice([1, 3, 8, 16, 32])
        while rows * heads * dim > 8192 * 32 * 128:
            rows = rows // 2 + 1
        c.pop("kv_heads"), c.pop("page")
        return dict(c, type=rng.choice(["f16", "bf16", "f32"]), rows=rows, heads=heads, positions=_log(rng, 100, 1000000),
                    **rope)
    if op == "fork":
        return dict(c, layers=rng.randint(1, 10), kv_heads=rng.choice([1, 2, 4]), length=_log(rng, 1, 20000),
                    children=_log(rng, 1, 16))
    if op == "compact":
        layers = rng.randint(1, 10)
        most = (256 * 10 * 2 * 256 * 64) // (layers * kv * dim * c["page"])
        return dict(c, layers=layers, pages=_log(rng, 1, max(2, min(most, 2000))))
    c["q_heads"] = kv * group
    n = _log(rng, 1, 64)
    tokens = 4096 if op == "attend" else 8192
    longest = _log(rng, 1, 131072)
    counts, lens = [], []
    for i in range(n):
        new = 1 if rng.random() < 0.6 else _log(rng, 1, max(2, tokens // n))
        counts.append(new)
        lens.append(new + (0 if rng.random() < 0.1 else _log(rng, 1, longest)))

    def too_much():
        scores = n * kv * group * max(counts) * max(lens)  # what the padded plain form holds
        cached = n * max(lens) * kv * dim
        rows = sum(counts) * kv * (group + 2) * dim
        return (scores > 32 * 4096 * 4096 or cached > 64 * 8001 * 4 * 128 or rows > 8192 * 40 * 128
                or sum(lens) * kv * dim > 64 * 4001 * 4 * 128 or scores * dim > 32 * 4096 * 2048 * 128)

    while too_much():
        k = max(range(n), key=lambda i: lens[i])
        counts[k], old = counts[k] // 2 + 1 if counts[k] > 2 else counts[k], lens[k] - counts[k]
        lens[k] = counts[k] + old // 2
        j = max(range(n), key=lambda i: counts[i])
        if counts[j] > 2:
            counts[j], lens[j] = counts[j] // 2 + 1, lens[j] - counts[j] + counts[j] // 2 + 1
    c.update(counts=" ".join(map(str, counts)), lens=" ".join(map(str, lens)))
    if op == "append":
        return dict(c, **rope)
    return dict(c, window=rng.choice([0, 0, 0, 128, 513, 4096]), sinks=rng.random() < 0.3, gate=rng.random() < 0.3)


def _batch(case):
    """(new tokens, positions with them) of each sequence."""
    counts = [int(a) for w in case["counts"].split() for a in [w.split("x")[0]] * int((w.split("x") + ["1"])[1])]
    w = case["lens"].split()
    if w[0] == "log":  # lengths spread over a range, in no order
        lo, hi, n = int(w[1]), int(w[2]), len(counts)
        lens = [int(lo * (hi / lo) ** (((i * 29) % n) / max(1, n - 1))) for i in range(n)]
    else:
        lens = [int(x) for x in w]
    return counts, lens


def _turns(counts, lens):
    """The positions each sequence grew by in each of the turns the cache was written in before the batch."""
    upto = [[(n - c) * k // TURNS for c, n in zip(counts, lens)] for k in range(TURNS + 1)]
    return [[b - a for a, b in zip(x, y)] for x, y in zip(upto, upto[1:])]


def _tables(counts, lens, page):
    """Page numbers by sequence, taken lowest first, turn by turn, then for the batch."""
    at, have, tables = 0, [0] * len(lens), [[] for _ in lens]
    for grown in _turns(counts, lens) + [counts]:
        for b, g in enumerate(grown):
            have[b] += g
            while len(tables[b]) * page < have[b]:
                tables[b].append(at)
                at += 1
    return tables, at


def work(case):
    b = 4 if case["type"] == "f32" else 2
    d = case["dim"]
    if case["op"] == "rotate":
        n = case["rows"] * case["heads"]
        return dict(bytes=2 * n * d * b + 4 * case["rows"], flops=3 * n * case["rot"])
    if case["op"] == "fork":
        copies = case["children"] if case["length"] % case["page"] else 0
        page = case["layers"] * 2 * case["kv_heads"] * case["page"] * d * b
        return dict(bytes=(copies + (copies > 0)) * page + 4 * case["children"], flops=0)
    if case["op"] == "compact":
        return dict(bytes=4 * case["pages"] * case["layers"] * 2 * case["kv_heads"] * case["page"] * d * b, flops=0)
    counts, lens = _batch(case)
    tokens = sum(counts)
    if case["op"] == "append":
        rows = tokens * (case["q_heads"] + 2 * case["kv_heads"])
        return dict(bytes=2 * rows * d * b, flops=3 * tokens * (case["q_heads"] + case["kv_heads"]) * case["rot"])
    keys = pairs = 0
    for c, n in zip(counts, lens):
        w = case["window"] or n
        keys += n - max(0, n - c + 1 - w)
        pairs += sum(min(w, n - c + t + 1) for t in range(c))
    moved = 2 * keys * case["kv_heads"] * d + (3 if case["gate"] else 2) * tokens * case["q_heads"] * d
    return dict(bytes=moved * b, flops=4 * pairs * case["q_heads"] * d)


def _rope(case):
    return dict(dim=case["rot"], layout=case["layout"], scaling=case["scaling"], base=case["base"],
                factor=case["factor"], original=case["original"])


def _natural(kv, layer):
    """A layer's K and V pages with the position before the head, from the layout that the library documents."""
    k, v = kv.pages(layer, 0), kv.pages(layer, 1)
    p, h, blocks, four, d, eight = v.shape
    return k.permute(0, 2, 4, 1, 3, 5), v.view(p, h, blocks, four, d, 2, 4).permute(0, 2, 5, 3, 6, 1, 4)


def _shaped(pool, which):
    """A plain pool [page][position][head][dim] in the shape of _natural()."""
    p, n, h, d = pool.shape
    return pool.view(p, n // 16, 16, h, d // 8, 8) if which == 0 else pool.view(p, n // 32, 2, 4, 4, h, d)


def _inputs(case, seed):
    """The tensors of a case, from the seed alone, and what its batch looks like."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = TYPES[case["type"]]

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda").to(t)

    d = case["dim"]
    if case["op"] == "rotate":
        pos = torch.randint(0, case["positions"], (case["rows"],), generator=g, device="cuda", dtype=torch.int32)
        return dict(x=normal(case["rows"], case["heads"], d), pos=pos)
    if case["op"] in ("fork", "compact"):
        n = case["pages"] if case["op"] == "compact" else -(-case["length"] // case["page"])
        total = 3 * n if case["op"] == "compact" else n + case["children"]
        return dict(n=n, total=total, pool=normal(case["layers"], 2, total, case["kv_heads"] * case["page"] * d))
    counts, lens = _batch(case)
    tables, total = _tables(counts, lens, case["page"])
    tokens = sum(counts)
    s = dict(counts=counts, lens=lens, tables=tables, tokens=tokens, q=normal(tokens, case["q_heads"], d),
             k_pool=normal(total, case["page"], case["kv_heads"], d),
             v_pool=normal(total, case["page"], case["kv_heads"], d))
    if case["op"] == "append":
        # k and v side by side, as the projection that makes both leaves them
        s["kv"] = normal(tokens, 2 * case["kv_heads"], d)
        s["k"], s["v"] = s["kv"][:, :case["kv_heads"]], s["kv"][:, case["kv_heads"]:]
    else:
        s["sinks"] = torch.randn(case["q_heads"], generator=g, device="cuda") if case["sinks"] else None
        s["gate"] = normal(tokens, case["q_heads"], d) if case["gate"] else None
    return s


def prepare(case, seed):
    s = dict(_inputs(case, seed), case=case, op=case["op"])
    if own:
        return _prepare_own(case, s)
    if case["op"] in ("attend", "append"):
        counts, lens = s["counts"], s["lens"]
        dev, most = "cuda", max(lens) // case["page"] + 1
        s["table"] = torch.tensor([t + [0] * (most - len(t)) for t in s["tables"]], device=dev)
        s["len"] = torch.tensor(lens, device=dev)
        s["count"] = torch.tensor(counts, device=dev)
        s["seq"] = torch.repeat_interleave(torch.arange(len(counts), device=dev), s["count"])
        first = torch.cumsum(s["count"], 0) - s["count"]
        s["turn"] = torch.arange(s["tokens"], device=dev) - first[s["seq"]]
        s["pos"] = (s["len"] - s["count"])[s["seq"]] + s["turn"]
    if case["op"] == "compact":
        s["at"] = s["n"]
    return s


def _prepare_own(case, s):
    from mechta_amd import paged
    if case["op"] == "rotate":
        return dict(s, rope=paged.Rope(**_rope(case)))
    fmt = {"f16": paged.F16, "bf16": paged.BF16}[case["type"]]
    if case["op"] in ("fork", "compact"):
        kv = paged.PagedKv(layers=case["layers"], q_heads=case["kv_heads"], kv_heads=case["kv_heads"],
                           head_dim=case["dim"], pages=s["total"], page=case["page"], seqs=20, ctx=262144, fmt=fmt)
        for layer in range(case["layers"]):
            for which in (0, 1):
                kv.pages(layer, which).copy_(s["pool"][layer, which].view(kv.pages(layer, which).shape))
        if case["op"] == "fork":
            kv.reserve([0], [case["length"]])
        else:  # slot 1 holds the pages below the conversation in slot 0
            kv.reserve([1], [s["n"] * case["page"]])
            kv.reserve([0], [s["n"] * case["page"]])
        del s["pool"]
        return dict(s, kv=kv)
    n = len(s["counts"])
    kv = paged.PagedKv(layers=1, q_heads=case["q_heads"], kv_heads=case["kv_heads"], head_dim=case["dim"],
                       pages=s["k_pool"].shape[0], page=case["page"], seqs=n, ctx=262144, fmt=fmt,
                       tokens=max(1, s["tokens"]), windows=[case.get("window", 0)],
                       rope=paged.Rope(**_rope(case)) if case["op"] == "append" else None)
    seqs = list(range(n))
    for grown in _turns(s["counts"], s["lens"]):
        kv.reserve(seqs, grown)
    kv.begin(seqs, s["counts"])
    for which, (view, pool) in enumerate(zip(_natural(kv, 0), (s["k_pool"], s["v_pool"]))):
        view.copy_(_shaped(pool, which))
    del s["k_pool"], s["v_pool"]
    return dict(s, kv=kv)


# ---- plain forms ----

def _angles(case, pos):
    """cos and sin of each row's angles, [rows, 1, rot / 2], amplitude included; angles in 64 bits."""
    r, base, f, n = case["rot"], case["base"], case["factor"], case["original"]
    i = torch.arange(r // 2, device=pos.device, dtype=torch.float64)
    amp = 1.0
    if case["scaling"] == "ntk":
        base = base * f ** (r / (r - 2))
    th = base ** (-2 * i / r)
    if case["scaling"] == "linear":
        th = th / f
    if case["scaling"] == "yarn":
        low, high = (r * math.log(n / (turns * 2 * math.pi)) / (2 * math.log(base)) for turns in (32, 1))
        low, high = max(math.floor(low), 0), min(math.ceil(high), r - 1)
        ramp = ((i - low) / max(high - low, 0.001)).clamp(0, 1)
        th = th / f * ramp + th * (1 - ramp)
        amp = 0.1 * math.log(f) + 1
    if case["scaling"] == "bands":
        s = ((n * th / (2 * math.pi) - 1) / (4 - 1)).clamp(0, 1)
        th = (1 - s) * th / f + s * th
    a = pos.double()[:, None, None] * th
    return (amp * a.cos()).float(), (amp * a.sin()).float()


def _rotated(case, x, cos, sin):
    """x [rows, heads, dim] rotated, in 32 bits, rounded once."""
    r, y = case["rot"], x.float()
    if case["layout"] == "half":
        a, b = y[..., :r // 2], y[..., r // 2:r]
        z = torch.cat((a * cos - b * sin, b * cos + a * sin, y[..., r:]), -1)
    else:
        a, b = y[..., 0:r:2], y[..., 1:r:2]
        z = torch.cat((torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2), y[..., r:]), -1)
    return z.to(x.dtype)


def _append(s):
    case = s["case"]
    cos, sin = _angles(case, s["pos"])
    page, at = s["table"][s["seq"], s["pos"] // case["page"]], s["pos"] % case["page"]
    s["k_pool"][page, at] = _rotated(case, s["k"], cos, sin)
    s["v_pool"][page, at] = s["v"]
    return dict(q=_rotated(case, s["q"], cos, sin), k=_shaped(s["k_pool"], 0), v=_shaped(s["v_pool"], 1))


def _attend(s):
    case = s["case"]
    h, d = case["kv_heads"], case["dim"]
    g, n, most = case["q_heads"] // h, len(s["lens"]), max(s["counts"])
    k, v = (s[p][s["table"]].flatten(1, 2).permute(0, 2, 1, 3).float() for p in ("k_pool", "v_pool"))
    q = torch.zeros(n, most, h, g, d, device="cuda")
    q[s["seq"], s["turn"]] = s["q"].view(-1, h, g, d).float()
    q = q.permute(0, 2, 1, 3, 4).reshape(n, h, most * g, d)
    score = (torch.matmul(q, k.transpose(2, 3).contiguous()) / math.sqrt(d)).view(n, h, most, g, -1)
    at = torch.arange(k.shape[2], device="cuda")
    pos = (s["len"] - s["count"])[:, None] + torch.arange(most, device="cuda")
    seen = at <= pos[:, :, None]
    if case["window"]:
        seen &= at > pos[:, :, None] - case["window"]
    score.masked_fill_(~seen[:, None, :, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    if s["sinks"] is not None:
        sink = s["sinks"].view(1, h, 1, g, 1)
        top = torch.maximum(top, sink)
    score.sub_(top).exp_()
    total = score.sum(-1, keepdim=True)
    if s["sinks"] is not None:
        total = total + torch.exp(sink - top)
    out = torch.matmul(score.view(n, h, most * g, -1), v).view(n, h, most, g, d) / total
    out = out.permute(0, 2, 1, 3, 4)[s["seq"], s["turn"]].reshape(-1, h * g, d)
    if s["gate"] is not None:
        out = out * torch.sigmoid(s["gate"].float())
    return out.to(s["q"].dtype)


def _pages_out(pools):
    return [p for layer in pools for p in layer]


def run(s):
    if own:
        return _run_own(s)
    case = s["case"]
    if s["op"] == "attend":
        return _attend(s)
    if s["op"] == "append":
        return _append(s)
    if s["op"] == "rotate":
        return _rotated(case, s["x"], *_angles(case, s["pos"]))
    pool, n = s["pool"], s["n"]
    if s["op"] == "fork":
        if case["length"] % case["page"]:
            pool[:, :, n:] = pool[:, :, n - 1:n]
        return _pages_out(pool)
    pool[:, :, :n] = pool[:, :, s["at"]:s["at"] + n]
    pool[:, :, 2 * n:] = pool[:, :, :n]
    s["at"] = 2 * n
    return dict(moved=n, pages=_pages_out(pool))


def _run_own(s):
    from mechta_amd import paged
    case = s["case"]
    if s["op"] == "attend":
        return s["kv"].attend(0, s["q"], sinks=s["sinks"], gate=s["gate"])
    if s["op"] == "append":
        q = s["kv"].append(0, s["k"], s["v"], s["q"])
        k, v = _natural(s["kv"], 0)
        return dict(q=q, k=k, v=v)
    if s["op"] == "rotate":
        return paged.rotate(s["x"], s["pos"], s["rope"])
    kv, n = s["kv"], s["n"]
    out = [kv.pages(layer, which).view(s["total"], -1) for layer in range(case["layers"]) for which in (0, 1)]
    if s["op"] == "fork":
        children = list(range(1, 1 + case["children"]))
        kv.fork([0] * len(children), children)
        kv.free(children)
        return out
    # the conversation in slot 0 moves down over the pages of slot 1; a second reader's copy of it is made above pages
    # that another sequence took meanwhile, and carries on in slot 0
    kv.free([1])
    moved = kv.compact()
    kv.reserve([2], [n * case["page"]])
    kv.copy([0], [3])
    kv.free([0, 2])
    kv.fork([3], [0])
    kv.free([3])
    kv.reserve([1], [n * case["page"]])
    return dict(moved=moved, pages=out)


# ---- the definition, in 64 bits ----

def _exact_rotated(case, x, pos):
    r = case["rot"]
    y = x.double().clone()
    p = pos.double().view(-1, 1)
    inv = []
    amp = 1.0
    for j in range(r // 2):
        f = case["base"] ** (-2.0 * j / r)
        if case["scaling"] == "linear":
            f /= case["factor"]
        elif case["scaling"] == "ntk":
            f = (case["base"] * case["factor"] ** (r / (r - 2.0))) ** (-2.0 * j / r)
        elif case["scaling"] == "yarn":
            def edge(turns):  # the pair that turns so many times over the original context
                return r * math.log(case["original"] / (turns * 2 * math.pi)) / (2 * math.log(case["base"]))
            lo, hi = max(math.floor(edge(32.0)), 0), min(math.ceil(edge(1.0)), r - 1)
            mix = min(1.0, max(0.0, (j - lo) / max(hi - lo, 0.001)))
            f = mix * f / case["factor"] + (1 - mix) * f
            amp = 1.0 + 0.1 * math.log(case["factor"])
        elif case["scaling"] == "bands":
            wave = 2 * math.pi / f
            if wave > case["original"]:
                f /= case["factor"]
            elif wave >= case["original"] / 4:
                mix = (case["original"] / wave - 1) / 3
                f = f * mix + (1 - mix) * f / case["factor"]
        inv.append(f)
    a = p * torch.tensor(inv, dtype=torch.float64, device=x.device)
    turn = torch.complex(amp * torch.cos(a), amp * torch.sin(a))[:, None, :]
    lo, hi = (slice(0, r // 2), slice(r // 2, r)) if case["layout"] == "half" else (slice(0, r, 2), slice(1, r, 2))
    z = torch.complex(y[..., lo], y[..., hi]) * turn
    y[..., lo], y[..., hi] = z.real, z.imag
    return y


def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "rotate":
        return _exact_rotated(case, s["x"], s["pos"])
    if case["op"] == "fork":
        pool, n = s["pool"].double(), s["n"]
        for c in range(case["children"] if case["length"] % case["page"] else 0):
            pool[:, :, n + c] = pool[:, :, n - 1]
        return [p for layer in pool for p in layer]
    if case["op"] == "compact":
        n = s["n"]
        return dict(moved=None, pages=[p[n:2 * n].repeat(3, 1).double() if i == 0 else
                                       torch.cat((p[n:2 * n],) * 3).double() for i, p in enumerate(s["pool"].flatten(0, 1))])
    h, d, page = case["kv_heads"], case["dim"], case["page"]
    g, first = case["q_heads"] // h, 0
    if case["op"] == "append":
        pos = torch.cat([torch.arange(n - c, n) for c, n in zip(s["counts"], s["lens"])]).cuda()
        k, kp, vp = _exact_rotated(case, s["k"], pos), s["k_pool"].double(), s["v_pool"].double()
        for c, n, table in zip(s["counts"], s["lens"], s["tables"]):
            flat = torch.tensor([table[p // page] * page + p % page for p in range(n - c, n)], device="cuda")
            kp.view(-1, h, d)[flat] = k[first:first + c]
            vp.view(-1, h, d)[flat] = s["v"][first:first + c].double()
            first += c
        return dict(q=_exact_rotated(case, s["q"], pos), k=_shaped(kp, 0), v=_shaped(vp, 1))
    out = torch.empty(s["tokens"], h * g, d, dtype=torch.float64, device="cuda")
    for c, n, table in zip(s["counts"], s["lens"], s["tables"]):
        k, v = (s[x][table].flatten(0, 1)[:n].double() for x in ("k_pool", "v_pool"))
        for t0 in range(0, c, 1024):  # so many of its tokens at a time
            t1 = min(c, t0 + 1024)
            p = torch.arange(n - c + t0, n - c + t1, device="cuda")[:, None]
            j = torch.arange(n, device="cuda")[None]
            hidden = (j > p) | (j <= p - (case["window"] or n + 1))
            for head in range(h * g):
                x = s["q"][first + t0:first + t1, head].double() @ k[:, head // g].T.contiguous() * d ** -0.5
                x[hidden] = -math.inf
                if case["sinks"]:  # one more key, whose value is zero
                    x = torch.cat((x, s["sinks"][head].double().expand(t1 - t0, 1)), 1)
                w = torch.softmax(x, 1)[:, :n]
                out[first + t0:first + t1, head] = w @ v[:, head // g]
        first += c
    return out * (1 / (1 + torch.exp(-s["gate"].double()))) if case["gate"] else out
