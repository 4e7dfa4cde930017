"""Timed cases of the paged K/V cache: what many sequences have in common is attended once, and what a sequence hardly
looks at is forgotten.

Three operators, each in its plain form (elementary torch operations in 32 bits, long sums in 64) and, with `own` set, as
a program calls the library (mechta_amd.paged):

- `shared`: attention of a batch whose sequences were forked off one prompt (and, in a tree, off each other): a batch begun
  as shared reads the positions that several sequences have in common once for all of them.
- `weigh`: the attention weights that the batch's tokens (all of them, or the last ones of each sequence) give to each
  position of the cache, summed over the tokens and over the query heads of a K/V head, added to what the position has
  accumulated before, which may fade.
- `evict`: of each sequence the first and the last positions are kept and, of those between, the ones of the largest
  accumulated weight, for each layer and K/V head by itself; K, V and the weights move together, in order. A pass does it to
  forks of conversations that stay whole.

Ranges: 1 to 64 sequences, 1 to 131,072 positions, 1 to 4,096 tokens a batch, head sizes 64, 128 and 256, 1 to 16 query
heads per K/V head, pages of 32 to 256 positions, f16 and bf16.
"""
import math

import torch

own = False

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # four samples of a short answer: one token each, the latency of a call
        dict(name="shared_4x_700", op="shared", type="f16", q_heads=16, kv_heads=2, dim=256, page=64, seqs=4, tokens=1,
             prompt=700, groups=1, middle=0, lo=1, hi=20, window=0, sinks=False, gate=True),
        # 64 samples of one long prompt generating side by side
        dict(name="shared_64x_8k", op="shared", type="bf16", q_heads=32, kv_heads=4, dim=128, page=64, seqs=64, tokens=1,
             prompt=8000, groups=1, middle=0, lo=10, hi=600, window=0, sinks=False, gate=False),
        # eight readers of one document, each verifying three drafted tokens
        dict(name="shared_verify4_8x_64k", op="shared", type="f16", q_heads=16, kv_heads=2, dim=256, page=128, seqs=8,
             tokens=4, prompt=65536, groups=1, middle=0, lo=100, hi=500, window=0, sinks=False, gate=True),
        # a tree: six users' conversations under one system prompt, eight samples of each, a sliding layer with sinks
        dict(name="shared_tree_window", op="shared", type="bf16", q_heads=32, kv_heads=8, dim=64, page=32, seqs=48, tokens=1,
             prompt=3001, groups=6, middle=700, lo=5, hi=300, window=2048, sinks=True, gate=False),
        # the step of one short conversation, every token counted: the latency of a call
        dict(name="weigh_1tok_300", op="weigh", type="f16", q_heads=16, kv_heads=2, dim=256, page=64, counts="1", lens="300",
             window=0, sinks=False, last=0, decay=1.0),
        # the step of 64 conversations generating side by side, lengths from a question to a document
        dict(name="weigh_64seq_decode", op="weigh", type="bf16", q_heads=32, kv_heads=4, dim=128, page=64, counts="1x64",
             lens="log 500 8001", window=0, sinks=False, last=0, decay=1.0),
        # a whole prompt, all of its tokens counted: the matrix units' case
        dict(name="weigh_prompt_4k", op="weigh", type="bf16", q_heads=32, kv_heads=4, dim=128, page=64, counts="4096",
             lens="4096", window=0, sinks=False, last=0, decay=0.0),
        # the last chunk of a long prompt: its last 32 tokens observe what the prompt's positions weigh
        dict(name="weigh_observe_16k", op="weigh", type="f16", q_heads=16, kv_heads=2, dim=256, page=64, counts="512",
             lens="16000", window=0, sinks=False, last=32, decay=0.0),
        # a sliding layer of a batch in which prompts arrive while others generate, with sinks; what was long ago fades
        dict(name="weigh_mixed_window", op="weigh", type="bf16", q_heads=32, kv_heads=4, dim=128, page=32,
             counts="700 256 33 1x12", lens="700 3001 97 1200 64 513 514 3999 2048 5 777 900 1500 4001 1", window=513,
             sinks=True, last=64, decay=0.9),
        # one conversation cut to half, one layer
        dict(name="evict_2k", op="evict", type="f16", kv_heads=2, dim=256, page=64, layers=1, lens="2000", keep=1024, first=4,
             recent=256),
        # a pool that has run full: 64 conversations cut to 1,500 positions each, the short ones left as they are
        dict(name="evict_64seq", op="evict", type="bf16", kv_heads=4, dim=128, page=64, layers=2, lens="64 log 1000 8001",
             keep=1500, first=4, recent=500),
        # a long document cut to a quarter, all layers
        dict(name="evict_64k", op="evict", type="f16", kv_heads=2, dim=256, page=64, layers=10, lens="65536", keep=16384,
             first=16, recent=4096),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["shared", "weigh", "evict"])
    kv, group, dim = rng.choice([1, 2, 3, 4, 8]), rng.choice([1, 2, 4, 5, 8, 16]), rng.choice([64, 128, 256])
    c = dict(op=op, type=rng.choice(["f16", "bf16"]), kv_heads=kv, dim=dim, page=rng.choice([32, 64, 128, 256]))
    if op == "evict":
        n, layers = _log(rng, 1, 64), rng.randint(1, 10)
        most = 65536 * 10 * 2 * 256 // (layers * kv * dim)  # positions in all
        lens = [_log(rng, 2, max(3, min(131072, most // n))) for _ in range(n)]
        keep = _log(rng, 1, max(lens))
        if sum(min(keep, x) for x in lens) * 4 > most:
            keep = max(1, most // (4 * n))
        first = rng.randint(0, keep // 4)
        return dict(c, layers=layers, lens=" ".join(map(str, lens)), keep=keep, first=first,
                    recent=rng.randint(0, (keep - first) // 2))
    c.update(q_heads=kv * group, window=rng.choice([0, 0, 0, 128, 513, 4096]), sinks=rng.random() < 0.3)
    if op == "shared":
        n, tokens = _log(rng, 2, 64), rng.choice([1, 1, 1, 2, 4, 7])
        groups = rng.choice([1, 1, rng.randint(1, n)])
        prompt, middle, hi = _log(rng, 16, 65536), _log(rng, 1, 4000) if groups > 1 else 0, _log(rng, 1, 2000)
        while n * (prompt + middle + hi + tokens) * kv * dim > 8 * 66000 * 2 * 256:  # what the padded plain form gathers
            prompt, middle, hi, n = prompt * 3 // 4 + 1, middle * 3 // 4, hi * 3 // 4 + 1, max(2, n * 7 // 8)
            groups = min(groups, n)
        return dict(c, seqs=n, tokens=tokens, prompt=prompt, groups=groups, middle=middle, lo=1, hi=hi, gate=rng.random() < 0.3)
    n, longest, last = _log(rng, 1, 64), _log(rng, 1, 131072), rng.choice([0, 0, 0, 1, 32, 64])
    counts, lens = [], []
    for _ in range(n):
        new = 1 if rng.random() < 0.6 else _log(rng, 1, max(2, 4096 // n))
        counts.append(new)
        lens.append(new + (0 if rng.random() < 0.1 else _log(rng, 1, longest)))

    def too_much():
        rows = max(min(x, last or x) for x in counts)
        scores = n * kv * group * rows * max(lens)  # what the padded plain form holds
        return (scores > 32 * 4096 * 4096 or scores * dim > 32 * 4096 * 4096 * 128
                or n * max(lens) * kv * dim > 64 * 8001 * 4 * 128 or sum(lens) * kv * dim > 64 * 4001 * 4 * 128)

    while too_much():
        k = max(range(n), key=lambda i: lens[i])
        counts[k], old = counts[k] // 2 + 1 if counts[k] > 2 else counts[k], lens[k] - counts[k]
        lens[k] = counts[k] + old // 2
        j = max(range(n), key=lambda i: counts[i])
        if counts[j] > 2:
            counts[j], lens[j] = counts[j] // 2 + 1, lens[j] - counts[j] + counts[j] // 2 + 1
    return dict(c, counts=" ".join(map(str, counts)), lens=" ".join(map(str, lens)), last=last,
                decay=rng.choice([0.0, 0.5, 0.9, 1.0, 1.0]))


def _spread(lo, hi, n):
    """Lengths spread over a range, in no order."""
    return [int(lo * (hi / lo) ** (((i * 29) % n) / max(1, n - 1))) for i in range(n)]


def _lens(text, n=None):
    w = text.split()
    if "log" in w:
        k = w.index("log")
        return _spread(int(w[k + 1]), int(w[k + 2]), n or int(w[0]))
    return [int(x) for x in w]


def _counts(text):
    return [int(a) for w in text.split() for a in [w.split("x")[0]] * int((w.split("x") + ["1"])[1])]


class _Family:
    """Page lists as the library takes them: pages lowest number first, forks share full pages."""

    def __init__(self, n, page):
        self.page, self.at, self.tables, self.lens, self.copies = page, 0, [[] for _ in range(n)], [0] * n, []

    def take(self):
        self.at += 1
        return self.at - 1

    def grow(self, seqs, counts):
        for s, c in zip(seqs, counts):
            self.lens[s] += c
            while len(self.tables[s]) * self.page < self.lens[s]:
                self.tables[s].append(self.take())

    def fork(self, src, dst):
        for a, b in zip(src, dst):
            full = self.lens[a] // self.page
            self.tables[b], self.lens[b] = self.tables[a][:full], self.lens[a]
            if self.lens[a] % self.page:
                self.tables[b].append(self.take())
                self.copies.append((self.tables[a][full], self.tables[b][full], self.lens[a] % self.page))


def _grown(case):
    """The steps in which a shared batch's sequences came to be: ("grow", sequences, counts) and ("fork", from, to)."""
    n, g = case["seqs"], case["groups"]
    own_parts = _spread(case["lo"], case["hi"], n)
    steps = [("grow", [0], [case["prompt"]]), ("fork", [0] * (g - 1), list(range(1, g)))]
    if g > 1:
        steps.append(("grow", list(range(g)), [case["middle"]] * g))
    steps.append(("fork", [s % g for s in range(g, n)], list(range(g, n))))
    steps.append(("grow", list(range(n)), own_parts))
    return [s for s in steps if s[1]], [case["tokens"]] * n


def _batch(case):
    """(new tokens, positions with them, page tables, pages, copied pages) of the batch."""
    if case["op"] == "shared":
        steps, counts = _grown(case)
        f = _Family(case["seqs"], case["page"])
        for what, a, b in steps:
            (f.grow if what == "grow" else f.fork)(a, b)
        f.grow(list(range(case["seqs"])), counts)
        return counts, f.lens, f.tables, f.at, f.copies
    if case["op"] == "weigh":
        counts = _counts(case["counts"])
        lens = _lens(case["lens"], len(counts))
    else:
        lens = _lens(case["lens"])
        counts = [0] * len(lens)
    f = _Family(len(lens), case["page"])
    for k in range(4):  # written in turns, so that pages lie scattered
        f.grow(range(len(lens)), [(n - c) * (k + 1) // 4 - (n - c) * k // 4 for c, n in zip(counts, lens)])
    f.grow(range(len(lens)), counts)
    return counts, f.lens, f.tables, f.at, f.copies


def _cut(case):
    """Page tables of the forks before and after the eviction, pages in all, and the pages that the forks copied."""
    _, lens, tables, total, _ = _batch(case)
    n = len(lens)
    f = _Family(2 * n, case["page"])
    f.at, f.tables[:n], f.lens[:n] = total, tables, lens
    f.fork(range(n), range(n, 2 * n))
    after = list(f.tables[n:])
    for s in range(n):
        if lens[s] > case["keep"]:
            after[s] = [f.take() for _ in range(-(-case["keep"] // case["page"]))]
    return after, f.at, f.copies


def work(case):
    d, h = case["dim"], case["kv_heads"]
    counts, lens, tables, _, _ = _batch(case)
    if case["op"] == "evict":
        kept = sum(case["keep"] for n in lens if n > case["keep"])
        read = sum(n for n in lens if n > case["keep"])
        return dict(bytes=case["layers"] * h * (kept * (2 * 2 * d * 2 + 4) + read * 4), flops=0)
    w, pairs, seen, keys = case["window"], 0, set(), 0
    last = case.get("last", 0)
    for s, (c, n) in enumerate(zip(counts, lens)):
        m = min(c, last or c)
        pairs += sum(min(w or n, n - m + t + 1) for t in range(m))
        if m:
            lo = max(0, n - m + 1 - w) if w else 0
            keys += n - lo
            for k in range(lo // case["page"], len(tables[s])):  # pages that several sequences have are read once
                at = range(max(lo, k * case["page"]), min(n, (k + 1) * case["page"]))
                seen.add((tables[s][k], at.start % case["page"], len(at)))
    by_page = {}
    for page, at, size in seen:
        a, b = by_page.get(page, (at, at + size))
        by_page[page] = (min(a, at), max(b, at + size))
    distinct, tokens = sum(b - a for a, b in by_page.values()), sum(min(c, last or c) for c in counts)
    if case["op"] == "shared":
        moved = 2 * distinct * h * d + (3 if case["gate"] else 2) * tokens * case["q_heads"] * d
        return dict(bytes=2 * moved, flops=4 * pairs * case["q_heads"] * d)
    touched = (keys if case["decay"] == 1 else sum(lens)) * (1 if case["decay"] == 0 else 2)
    return dict(bytes=2 * (keys * h + tokens * case["q_heads"]) * d + 4 * touched * h, flops=2 * pairs * case["q_heads"] * d)


def _inputs(case, seed):
    """The tensors of a case, from the seed alone, and what its batch looks like."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    t, d, h = TYPES[case["type"]], case["dim"], case["kv_heads"]

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda").to(t)

    counts, lens, tables, total, copies = _batch(case)
    s = dict(counts=counts, lens=lens, tables=tables, tokens=sum(counts))
    if case["op"] == "evict":
        s["after"], total, copies = _cut(case)
        s["copies"] = copies
        s["k_pool"], s["v_pool"] = (normal(case["layers"], total, case["page"], h, d) for _ in range(2))
        # a few positions weigh much, many alike, some nothing yet
        w = torch.randn((case["layers"], len(lens), h, max(lens)), generator=g, device="cuda").mul_(2).exp_()
        w = torch.where(w < 0.1, torch.zeros_like(w), torch.where(w < 0.5, (w * 64).round_() / 64, w))
        here = torch.arange(max(lens), device="cuda") < torch.tensor(lens, device="cuda")[:, None, None]
        s["weights"] = w * here
        return s
    s["k_pool"], s["v_pool"] = (normal(total, case["page"], h, d) for _ in range(2))
    for a, b, upto in copies:
        for p in ("k_pool", "v_pool"):
            s[p][b, :upto] = s[p][a, :upto]
    s["q"] = normal(s["tokens"], case["q_heads"], d)
    s["sinks"] = torch.randn(case["q_heads"], generator=g, device="cuda") if case["sinks"] else None
    s["gate"] = normal(s["tokens"], case["q_heads"], d) if case.get("gate") else None
    if case["op"] == "weigh":
        # as some steps before have left them
        s["weights"] = torch.rand((len(lens), h, max(lens)), generator=g, device="cuda") * 16 / max(lens)
        del s["v_pool"]
    return s


def _natural(kv, layer, which):
    """A layer's K or V pages with the position before the head, from the layout that the library documents."""
    x = kv.pages(layer, which)
    if which == 0:
        return x.permute(0, 2, 4, 1, 3, 5)
    p, h, blocks, four, d, eight = x.shape
    return x.view(p, h, blocks, four, d, 2, 4).permute(0, 2, 5, 3, 6, 1, 4)


def _shaped(pool, which):
    """A plain pool [page][position][head][dim] in the shape of _natural()."""
    p, n, h, d = pool.shape
    return pool.view(p, n // 16, 16, h, d // 8, 8) if which == 0 else pool.view(p, n // 32, 2, 4, 4, h, d)


def prepare(case, seed):
    s = dict(_inputs(case, seed), case=case, op=case["op"])
    if own:
        return _prepare_own(case, s)
    dev, page = "cuda", case["page"]

    def padded(tables):
        most = max(map(len, tables))
        return torch.tensor([t + [0] * (most - len(t)) for t in tables], device=dev)

    s["table"], s["len"] = padded(s["tables"]), torch.tensor(s["lens"], device=dev)
    if case["op"] == "evict":
        n, total = len(s["lens"]), s["k_pool"].shape[1]
        s["from"], s["to"] = (torch.tensor([c[i] for c in s["copies"]], device=dev, dtype=torch.long) for i in (0, 1))
        cut = [i for i in range(n) if s["lens"][i] > case["keep"]]
        s["cut"] = torch.tensor(cut, device=dev, dtype=torch.long)
        at = torch.arange(case["keep"], device=dev)
        s["new"] = padded([s["after"][i] for i in cut])[:, at // page] * page + at % page if cut else None
        s["first_new"] = total - sum(-(-case["keep"] // page) for _ in cut) - len(s["copies"])
        s["kept"] = s["weights"].clone()
        return s
    last = case.get("last", 0)
    counted = [min(c, last or c) for c in s["counts"]]
    s["count"] = torch.tensor(counted, device=dev)
    s["seq"] = torch.repeat_interleave(torch.arange(len(counted), device=dev), s["count"])
    first = torch.cumsum(torch.tensor(s["counts"], device=dev), 0) - s["count"]  # of the counted tokens in the batch
    before = torch.cumsum(s["count"], 0) - s["count"]
    s["turn"] = torch.arange(sum(counted), device=dev) - before[s["seq"]]
    s["row"] = first[s["seq"]] + s["turn"]
    s["most"] = max(counted)
    return s


def _prepare_own(case, s):
    from mechta_amd import paged
    fmt = {"f16": paged.F16, "bf16": paged.BF16}[case["type"]]
    n, h, page = len(s["lens"]), case["kv_heads"], case["page"]
    layers, seqs = case.get("layers", 1), list(range(n))
    pages = s["k_pool"].shape[1 if case["op"] == "evict" else 0]
    kv = paged.PagedKv(layers=layers, q_heads=case.get("q_heads", h), kv_heads=h, head_dim=case["dim"], pages=pages, page=page,
                       seqs=2 * n if case["op"] == "evict" else n, ctx=max(s["lens"]), fmt=fmt, tokens=max(1, s["tokens"]),
                       windows=[case.get("window", 0)] * layers,
                       weigh_last=None if case["op"] == "shared" else case.get("last", 0))
    if case["op"] == "shared":
        for what, a, b in _grown(case)[0]:
            (kv.reserve if what == "grow" else kv.fork)(a, b)
        kv.begin(seqs, s["counts"], shared=True)
    else:
        for k in range(4):
            kv.reserve(seqs, [(m - c) * (k + 1) // 4 - (m - c) * k // 4 for c, m in zip(s["counts"], s["lens"])])
    if case["op"] == "weigh":
        kv.begin(seqs, s["counts"])
        kv.weights(0).copy_(s["weights"])
        _natural(kv, 0, 0).copy_(_shaped(s.pop("k_pool"), 0))
        return dict(s, kv=kv, out=kv.weights(0))
    for layer in range(layers):
        for which, name in enumerate(("k_pool", "v_pool")):
            pool = s[name][layer] if case["op"] == "evict" else s[name]
            _natural(kv, layer, which).copy_(_shaped(pool, which))
        if case["op"] == "evict":
            kv.weights(layer)[:n].copy_(s["weights"][layer])
    del s["k_pool"], s["v_pool"]
    if case["op"] == "evict":
        cut = sum(m > case["keep"] for m in s["lens"])
        first_new = pages - cut * -(-case["keep"] // page) - len(s["copies"])
        s["out"] = dict(k=[_natural(kv, layer, 0)[first_new:] for layer in range(layers)],
                        v=[_natural(kv, layer, 1)[first_new:] for layer in range(layers)],
                        weights=[kv.weights(layer)[n:, :, :case["keep"]] for layer in range(layers)])
        s["forks"] = list(range(n, 2 * n))
        del s["weights"]
    return dict(s, kv=kv)


# ---- plain forms ----

def _scores(s):
    """exp(scores - top) of the counted tokens [sequence, head, token x group, position], and its sums with the sink."""
    case = s["case"]
    h, d, n, most = case["kv_heads"], case["dim"], len(s["lens"]), s["most"]
    g = case["q_heads"] // h
    k = s["k_pool"][s["table"]].flatten(1, 2).permute(0, 2, 3, 1).float().contiguous()
    q = torch.zeros(n, most, h, g, d, device="cuda")
    q[s["seq"], s["turn"]] = s["q"][s["row"]].view(-1, h, g, d).float()
    q = q.permute(0, 2, 1, 3, 4).reshape(n, h, most * g, d)
    score = (torch.matmul(q, k) / math.sqrt(d)).view(n, h, most, g, -1)
    del k, q
    at = torch.arange(score.shape[-1], device="cuda")
    pos = (s["len"] - s["count"])[:, None] + torch.arange(most, device="cuda")
    seen = (at <= pos[:, :, None]) & (torch.arange(most, device="cuda")[:, None] < s["count"][:, None, None])
    if case["window"]:
        seen &= at > pos[:, :, None] - case["window"]
    score.masked_fill_(~seen[:, None, :, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    if s["sinks"] is not None:
        sink = s["sinks"].view(1, h, 1, g, 1)
        top = torch.maximum(top, sink)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)  # (tokens that a shorter sequence does not have)
    score.sub_(top).exp_()
    total = score.sum(-1, keepdim=True)
    if s["sinks"] is not None:
        total = total + torch.exp(sink - top)
    return score, total


def _shared(s):
    case = s["case"]
    n, h, most, d = len(s["lens"]), case["kv_heads"], s["most"], case["dim"]
    g = case["q_heads"] // h
    score, total = _scores(s)
    v = s["v_pool"][s["table"]].flatten(1, 2).permute(0, 2, 1, 3).float().contiguous()
    out = torch.matmul(score.view(n, h, most * g, -1), v).view(n, h, most, g, d) / total
    out = out.permute(0, 2, 1, 3, 4)[s["seq"], s["turn"]].reshape(-1, h * g, d)
    if s["gate"] is not None:
        out = out * torch.sigmoid(s["gate"].float())
    return out.to(s["q"].dtype)


def _weigh(s):
    score, total = _scores(s)
    score.div_(torch.where(total == 0, torch.ones_like(total), total))
    new = score.flatten(2, 3).sum(2, dtype=torch.float64)[..., :s["weights"].shape[-1]]
    here = torch.arange(s["weights"].shape[-1], device="cuda") < s["len"][:, None, None]
    here = here & (s["count"] > 0)[:, None, None]
    before = s["case"]["decay"] * s["weights"].double() if s["case"]["decay"] else 0
    s["weights"] = torch.where(here, (before + new).float(), s["weights"])
    return s["weights"]


def _evict(s):
    case = s["case"]
    keep, first, recent, page = case["keep"], case["first"], case["recent"], case["page"]
    layers, n, h, most = s["weights"].shape
    if len(s["from"]):  # the forks' partly filled last pages
        for p in ("k_pool", "v_pool"):
            s[p][:, s["to"]] = s[p][:, s["from"]]
    s["kept"].copy_(s["weights"])
    if len(s["cut"]):
        w = s["weights"][:, s["cut"]].clone()
        at, end = torch.arange(most, device="cuda"), s["len"][s["cut"]][:, None, None]
        w.masked_fill_((at < first) | (at >= end - recent), math.inf)
        w.masked_fill_(at >= end, -1.0)
        order = w.sort(dim=-1, descending=True, stable=True).indices[..., :keep].sort(-1).values  # [layer, sequence, head, keep]
        old = s["table"][s["cut"]][None, :, None].expand(layers, -1, h, -1).gather(3, order // page) * page + order % page
        layer, head = (torch.arange(x, device="cuda") for x in (layers, h))
        for p in ("k_pool", "v_pool"):
            rows = s[p].flatten(1, 2)  # [layer, page x position, head, dim]
            rows[layer[:, None, None, None], s["new"][None, :, None], head[None, None, :, None]] = \
                rows[layer[:, None, None, None], old, head[None, None, :, None]]
        s["kept"][:, s["cut"], :, :keep] = s["weights"][:, s["cut"]].gather(3, order)
    new = s["first_new"]
    return dict(k=[_shaped(x[new:], 0) for x in s["k_pool"]], v=[_shaped(x[new:], 1) for x in s["v_pool"]],
                weights=[x[..., :keep] for x in s["kept"]])


def run(s):
    case = s["case"]
    if own:
        if s["op"] == "shared":
            return s["kv"].attend(0, s["q"], sinks=s["sinks"], gate=s["gate"])
        if s["op"] == "weigh":
            s["kv"].weigh(0, s["q"], sinks=s["sinks"], decay=case["decay"])
            return s["out"]
        s["kv"].free(s["forks"])  # of the pass before
        s["kv"].fork(range(len(s["forks"])), s["forks"])
        s["kv"].evict(s["forks"], case["keep"], first=case["first"], recent=case["recent"])
        return s["out"]
    return _shared(s) if s["op"] == "shared" else _weigh(s) if s["op"] == "weigh" else _evict(s)


# ---- the definition, in 64 bits ----

def exact(case, seed):
    s = _inputs(case, seed)
    h, d, page, first = case["kv_heads"], case["dim"], case["page"], 0
    if case["op"] == "evict":
        kp, vp = s["k_pool"].double(), s["v_pool"].double()
        for a, b, _ in s["copies"]:
            kp[:, b], vp[:, b] = kp[:, a], vp[:, a]
        weights = [w.double().cpu() for w in s["weights"]]
        for i, n in enumerate(s["lens"]):
            if n <= case["keep"]:
                continue
            flat = torch.tensor([s["tables"][i][p // page] * page + p % page for p in range(n)])
            to = torch.tensor([s["after"][i][p // page] * page + p % page for p in range(case["keep"])], device="cuda")
            for layer, w in enumerate(weights):
                for head in range(h):
                    lo, hi = case["first"], n - case["recent"]
                    rank = torch.argsort(-w[i, head, lo:hi], stable=True)[:case["keep"] - case["first"] - case["recent"]]
                    kept = torch.cat((torch.arange(lo), lo + torch.sort(rank).values, torch.arange(hi, n)))
                    for pool in (kp, vp):
                        rows = pool[layer].view(-1, h, d)
                        rows[to, head] = rows[flat[kept].cuda(), head]
                    w[i, head, :len(kept)] = w[i, head, kept]
        new = kp.shape[1] - sum(-(-case["keep"] // page) for n in s["lens"] if n > case["keep"]) - len(s["copies"])
        return dict(k=[_shaped(x[new:], 0) for x in kp], v=[_shaped(x[new:], 1) for x in vp],
                    weights=[w[..., :case["keep"]] for w in weights])
    g = case["q_heads"] // h
    shared = case["op"] == "shared"
    out = torch.empty(s["tokens"], h * g, d, dtype=torch.float64, device="cuda") if shared else s["weights"].double()
    for i, (c, n, table) in enumerate(zip(s["counts"], s["lens"], s["tables"])):
        k = s["k_pool"][table].flatten(0, 1)[:n].double()
        v = s["v_pool"][table].flatten(0, 1)[:n].double() if shared else None
        m = min(c, case.get("last", 0) or c)
        if not shared and m:
            out[i, :, :n] *= case["decay"]
        for t0 in range(c - m, c, 1024):  # so many of its tokens at a time
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
                if shared:
                    out[first + t0:first + t1, head] = w @ v[:, head // g]
                else:
                    out[i, head // g, :n] += w.sum(0)
        first += c
    return out * (1 / (1 + torch.exp(-s["gate"].double()))) if shared and case["gate"] else out
