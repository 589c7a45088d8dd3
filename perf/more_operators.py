"""The operators around a serving step's attention: what is measured of them.

Three kinds of work. `chunk`: a chunk of a prompt (or a batch of chunks and single tokens) attending over a paged, quantised
cache that holds it already. `plan`: the pages that rejected drafts and finished requests held given back, and the next
step's page tables, starts, slots and positions made from the requests' lengths. `verify`: drafted tokens held against the
target's logits with given random numbers, the accepted path's moves within the cache.

The cache is two buffers, codes u8 [pages][kv heads][2][page * dim] and scales f32 [pages][kv heads][2][page], keys then
values. Token t of a page, dimension d, lies in the keys' block at
    (t / 16) * 16 dim + (d / 64) * 1024 + (t % 16) * 64 + d % 64
and in the values' at
    (t / 64) * 64 dim + d * 64 + (t % 16 / 4) * 16 + (t % 64 / 16) * 4 + t % 4.
i8 codes are q + 128, e4m3 codes are the type's bytes; each vector has a scale. A slot is its page times the page's length
plus its place in it."""

import math
import random

import torch

own = False

# attention of the two model sizes that the package is measured on: gated queries
SIZE_4B = {"heads": 16, "kv_heads": 4, "dim": 256, "gated": True}
SIZE_27B = {"heads": 24, "kv_heads": 4, "dim": 256, "gated": True}
# a grouped-query layer without gates
SIZE_GQA = {"heads": 32, "kv_heads": 8, "dim": 128, "gated": False}
VOCAB = 248320


def _chunk(name, fmt, size, seqs, lo, hi, tokens, page=256):
    return {"name": name, "what": "chunk", "fmt": fmt, **size, "page": page, "seqs": seqs, "len_lo": lo, "len_hi": hi,
            "tokens": tokens}


def _plan(name, seqs, page, lo, hi, tokens, tree, short):
    return {"name": name, "what": "plan", "seqs": seqs, "page": page, "len_lo": lo, "len_hi": hi, "tokens": tokens,
            "tree": tree, "short": short}


def _verify(name, seqs, tokens, vocab, tree, draft):
    return {"name": name, "what": "verify", "seqs": seqs, "tokens": tokens, "vocab": vocab, "tree": tree, "draft": draft}


def listed():
    return [
        # the smallest call: a short question
        _chunk("chunk_4b_65", "i8", SIZE_4B, 1, 0, 0, 65),
        # the first chunk of a prompt
        _chunk("chunk_27b_2048", "i8", SIZE_27B, 1, 0, 0, 2048),
        # the largest: a chunk in the middle of a long document
        _chunk("chunk_27b_2048_len30k", "e4m3", SIZE_27B, 1, 30001, 30001, 2048),
        # the short rest of a prompt after a very long shared prefix
        _chunk("chunk_27b_131_len120k", "i8", SIZE_27B, 1, 120000, 120000, 131),
        # a batch that mixes chunks of many lengths with single tokens
        _chunk("chunk_gqa_batch12", "e4m3", SIZE_GQA, 12, 10, 4000, 300, page=64),
        # one request, its next five tokens
        _plan("plan_1", 1, 256, 4090, 4090, 5, False, False),
        # a full server: many small trees, and more requests than pages
        _plan("plan_trees_1000", 1000, 64, 1, 6000, 8, True, True),
        # prompts that arrive together
        _plan("plan_prompts_16", 16, 256, 0, 30000, 2048, False, False),
        # one conversation: four drafted tokens
        _verify("verify_1x5", 1, 5, VOCAB, False, False),
        # the largest tree
        _verify("verify_tree64", 1, 64, VOCAB, True, False),
        # a batch of drafted chains with the drafts' probabilities
        _verify("verify_draft_12x5", 12, 5, VOCAB, False, True),
    ]


def _log(rng, lo, hi):
    return int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))


def draw(rng):
    what = rng.choice(("chunk", "chunk", "plan", "verify"))
    if what == "plan":
        tokens = rng.choice((1, 4, 8, 64, 500, 2000))
        seqs = _log(rng, 1, min(1000, 40000 // tokens))
        hi = _log(rng, 1, 40000)
        return {"what": what, "seqs": seqs, "page": rng.choice((64, 128, 256, 1024)), "len_lo": int(hi * rng.uniform(0.0, 1.0)),
                "len_hi": hi, "tokens": tokens, "tree": 1 < tokens <= 64 and rng.random() < 0.5, "short": rng.random() < 0.4}
    if what == "verify":
        tokens = rng.choice((1, 2, 3, 5, 8, 21, 64))
        draft = tokens > 1 and rng.random() < 0.5
        return {"what": what, "seqs": _log(rng, 1, 64 // tokens), "tokens": tokens, "vocab": _log(rng, 500, 250000),
                "tree": not draft and tokens > 2 and rng.random() < 0.6, "draft": draft}
    dim = rng.choice((64, 128, 256))
    kv_heads = rng.choice((1, 2, 4, 8))
    heads = kv_heads * rng.choice((1, 2, 3, 4, 5, 6, 8))
    seqs = rng.choice((1, 1, 2, 5, 11))
    tokens = _log(rng, 65, 2500 // seqs)
    hi = _log(rng, 10, min(130000, int(1.5e9) // (heads * seqs * tokens)))
    return {"what": what, "fmt": rng.choice(("i8", "e4m3")), "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "gated": rng.random() < 0.5, "page": rng.choice((64, 128, 256)), "seqs": seqs,
            "len_lo": rng.choice((0, int(hi * rng.uniform(0.0, 1.0)))), "len_hi": hi, "tokens": tokens}


# ---- inputs ---------------------------------------------------------------------------------------------------------


def _gen(seed, name):
    g = torch.Generator(device="cuda")
    g.manual_seed((seed * 1_000_003 + sum((i + 1) * ord(c) for i, c in enumerate(name))) & 0x7FFFFFFFFFFF)
    return g


def _dev(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


def _requests(c):
    """(cached tokens, new tokens) of each sequence: the same for every seed. Of four sequences and more, one has nothing
    new in this step, one nothing cached yet and one a single new token."""
    rng = random.Random("%s %s %s" % (c["seqs"], c["len_hi"], c["tokens"]))
    lo, hi = c["len_lo"], c["len_hi"]
    lens = [max(lo, min(hi, _log(rng, max(lo, 1), max(hi, 1)))) for _ in range(c["seqs"])]
    news = [_log(rng, 1, c["tokens"]) for _ in range(c["seqs"])]
    lens[0], news[0] = hi, c["tokens"]
    if c["seqs"] >= 4:
        news[1], lens[2], news[3] = 0, 0, 1
    return lens, news


def _left_over(c):
    """Pages that each sequence holds past its positions."""
    rng = random.Random("%s %s" % (c["seqs"], c["page"]))
    return [rng.choice((0, 0, 1, 2)) for _ in range(c["seqs"])]


def _drafted(c):
    """Tokens of each sequence that are verified."""
    rng = random.Random("%s %s %s" % (c["seqs"], c["tokens"], c["vocab"]))
    return [c["tokens"]] + [rng.randint(1, c["tokens"]) for _ in range(c["seqs"] - 1)]


def _tree(rng, n, tree):
    """Masks of the nodes that each node sees (itself and its ancestors): a chain, or parents at random."""
    masks = [1] if n else []
    for i in range(1, n):
        masks.append(masks[rng.randint(max(0, i - 6), i - 1) if tree else i - 1] | 1 << i)
    return masks


def _signed(u):
    return u - (1 << 64) if u >> 63 else u


def _starts(news):
    at = [0]
    for m in news:
        at.append(at[-1] + m)
    return at


def _prepare_chunk(c, g, seed):
    lens, news = _requests(c)
    rng = random.Random(seed)
    held = [-(-(a + b) // c["page"]) for a, b in zip(lens, news)]
    pages = sum(held) + 2
    order = list(range(pages))
    rng.shuffle(order)
    width = max(max(held), 1)
    table = [[order.pop() for _ in range(h)] for h in held]
    shape = (pages, c["kv_heads"], 2, c["page"] * c["dim"])
    values = torch.randn(shape, generator=g, device="cuda", dtype=torch.float16 if math.prod(shape) > 1 << 26 else torch.float32)
    if c["fmt"] == "i8":
        codes, size = ((values * 40).round_().clamp_(-127, 127) + 128).to(torch.uint8), 0.025
    else:
        codes, size = (values * 100).clamp_(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8), 0.01
    scales = torch.rand(shape[:3] + (c["page"],), generator=g, device="cuda") * size + 0.5 * size
    used = _dev([p for row in table for p in row], torch.int64)
    place = _dev([k for h in held for k in range(h)], torch.int64)
    total = _dev([a + b for a, b, h in zip(lens, news, held) for _ in range(h)], torch.int64)
    written = torch.zeros((pages, c["page"]), dtype=torch.bool, device="cuda")
    if len(used):
        written[used] = place[:, None] * c["page"] + torch.arange(c["page"], device="cuda") < total[:, None]
    # what no sequence has written is whatever the memory held
    scales = torch.where(written[:, None, None, :], scales, float("nan"))
    n = sum(news)
    strength = torch.rand((n, c["heads"], 1), generator=g, device="cuda") * 3 + 0.3  # flat and peaked heads
    q = (torch.randn((n, c["heads"], c["dim"]), generator=g, device="cuda") * strength).to(torch.bfloat16)
    gate = torch.randn(q.shape, generator=g, device="cuda").to(torch.bfloat16) if c["gated"] else None
    return {"codes": codes, "scales": scales, "start": _dev(_starts(news)), "len": _dev(lens), "n": n, "width": width,
            "table": _dev([row + [-1] * (width - len(row)) for row in table]), "q": q, "gate": gate, "out": torch.empty_like(q)}


def _prepare_plan(c, g, seed):
    lens, news = _requests(c)
    rng = random.Random(seed)
    page = c["page"]
    # what the last step left: some requests hold a page or more for tokens that were rejected
    held = [-(-a // page) + k for a, k in zip(lens, _left_over(c))]
    need = [max(0, -(-(a + m) // page) - -(-a // page)) if m else 0 for a, m in zip(lens, news)]
    spare = sum(h - -(-a // page) for h, a in zip(held, lens))
    left = max(0, int(sum(need) * 0.9) - spare) if c["short"] else sum(need) + 7
    order = list(range(sum(held) + left))
    rng.shuffle(order)
    width = max(max(h, -(-(a + m) // page)) for h, a, m in zip(held, lens, news)) + 1
    table = [[order.pop() for _ in range(h)] for h in held]
    pages, n = len(order) + sum(held), sum(news)
    tree_rng = random.Random(seed + 1)
    masks = [_signed(v) for m in news for v in _tree(tree_rng, m, True)] if c["tree"] else None
    empty = lambda k: torch.empty(max(k, 1), dtype=torch.int32, device="cuda")[:k]  # noqa: E731
    return {"pages": pages, "n": n, "width": width, "free": _dev(order + [-1] * (pages - len(order))), "n_free": _dev([len(order)]),
            "table": _dev([row + [-1] * (width - len(row)) for row in table]), "held": _dev(held), "len": _dev(lens),
            "add": _dev(news), "mask": _dev(masks, torch.int64) if c["tree"] else None, "start": empty(c["seqs"] + 1),
            "slots": empty(n), "pos": empty(n), "granted": empty(c["seqs"])}


def _prepare_verify(c, g, seed):
    b, v = c["seqs"], c["vocab"]
    rng = random.Random(seed)
    news = _drafted(c)
    n = sum(news)
    # heads that are sure and heads that are not: a favourite of each row above a bell of logits
    logits = torch.randn((n, v), generator=g, device="cuda") * 2.0
    favourite = torch.randint(0, v, (n, 3), generator=g, device="cuda")
    raise_by = torch.rand((n, 1), generator=g, device="cuda") * 12 + torch.tensor([8.0, 7.0, 6.0], device="cuda")
    logits.scatter_(1, favourite, raise_by)
    tokens, masks = torch.randint(0, v, (n,), generator=g, device="cuda"), []
    starts, likely = _starts(news), favourite.tolist()
    drafted = tokens.tolist()
    for k, a in zip(news, starts):
        mine = _tree(rng, k, c["tree"])
        children = [0] * k
        for i in range(1, k):
            parent = (mine[i] ^ 1 << i).bit_length() - 1
            # a node's children are the draft's best guesses in turn
            if children[parent] < 3 and rng.random() < 0.9:
                drafted[a + i] = likely[a + parent][children[parent]]
            children[parent] += 1
        masks += [_signed(x) for x in mine]
    draft = None
    if c["draft"]:
        draft = torch.softmax(logits * 0.9 + 0.3 * torch.randn((n, v), generator=g, device="cuda"), -1)
        picked = torch.multinomial(draft, 1, generator=g)[:, 0].tolist()
        drafted = [d if i in starts else picked[i - 1] for i, d in enumerate(drafted)]
    lens = [4000 + k * 37 % 1000 for k in range(b)]
    page = 256
    held = [-(-(a + k) // page) for a, k in zip(lens, news)]
    order = list(range(sum(held)))
    rng.shuffle(order)
    width = max(held)
    empty = lambda k: torch.empty(k, dtype=torch.int32, device="cuda")  # noqa: E731
    return {"n": n, "logits": logits, "tokens": _dev(drafted), "draft": draft, "page": page, "start": _dev(starts), "len": _dev(lens),
            "table": _dev([[order.pop() for _ in range(h)] + [-1] * (width - h) for h in held]),
            "mask": _dev(masks, torch.int64) if c["tree"] else None,
            # some requests want the likeliest token
            "temp": _dev([0.0 if i % 4 == 3 else rng.choice((0.6, 0.8, 1.0)) for i in range(b)], torch.float32),
            "u": torch.rand((n, 2), generator=g, device="cuda"), "next": empty(b), "count": empty(b), "emit": empty(n),
            "src": empty(n), "dst": empty(n), "new_len": empty(b)}


def prepare(case, seed):
    c = case
    made = {"chunk": _prepare_chunk, "plan": _prepare_plan, "verify": _prepare_verify}[c["what"]](c, _gen(seed, c["what"]), seed)
    return {"case": c, "kept": {}, **made}


# ---- the plain form -------------------------------------------------------------------------------------------------


def _history(c, s):
    """The sequences' keys and values from the cache, f32 [seqs][kv heads][positions][dim] each; pages that a sequence has
    not are taken from page 0."""
    b, w, j, d, p = c["seqs"], s["width"], c["kv_heads"], c["dim"], c["page"]
    table = s["table"].long().clamp(min=0)
    codes, scales = s["codes"][table], s["scales"][table]
    codes = codes.float() - 128 if c["fmt"] == "i8" else codes.view(torch.float8_e4m3fn).float()
    k = codes[:, :, :, 0].view(b, w, j, p // 16, d // 64, 16, 64).permute(0, 2, 1, 3, 5, 4, 6)
    v = codes[:, :, :, 1].view(b, w, j, p // 64, d, 4, 4, 4).permute(0, 2, 1, 3, 6, 5, 7, 4)
    at = scales.permute(3, 0, 2, 1, 4).reshape(2, b, j, w * p, 1)
    return k.reshape(b, j, w * p, d) * at[0], v.reshape(b, j, w * p, d) * at[1]


def _plain_chunk(c, s):
    b, j, d, m = c["seqs"], c["kv_heads"], c["dim"], c["tokens"]
    group = c["heads"] // j
    start, lens = s["start"].long(), s["len"].long()
    node = torch.arange(m, device="cuda")
    news = start[1:] - start[:-1]
    token = torch.where(node < news[:, None], start[:-1, None] + node, s["n"])  # [seqs][m], padded with a token of zeros
    q = s["q"].float()
    padded = torch.cat((q, torch.zeros_like(q[:1])))[token].view(b, m, j, group, d).permute(0, 2, 1, 3, 4)
    k, v = _history(c, s)
    fresh = torch.arange(k.shape[2], device="cuda") - lens[:, None]  # which of the chunk's tokens lies at a position
    held = (fresh < news[:, None])[:, None, :, None]
    k, v = torch.where(held, k, 0.0), torch.where(held, v, 0.0)
    scores = torch.matmul(padded.reshape(b, j, m * group, d) * d**-0.5, k.transpose(-1, -2)).view(b, j, m, group, -1)
    scores = scores.masked_fill_((fresh[:, None] > node[:, None])[:, None, :, None], float("-inf"))
    p = scores.sub_(scores.amax(-1, keepdim=True)).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(b, j, m * group, -1), v).view(b, j, m, group, d) / total
    o = o.permute(0, 2, 1, 3, 4).reshape(b * m, -1, d)[(node < news[:, None]).view(-1)]
    return {"out": (o * torch.sigmoid(s["gate"].float()) if c["gated"] else o).to(torch.bfloat16)}


def _slot(table, page, seq, position):
    return (table.long()[seq, position // page] * page + position % page).to(torch.int32)


def _plain_plan(c, s):
    page, width, b = c["page"], s["width"], c["seqs"]
    lens, add, place = s["len"].long(), s["add"].long(), torch.arange(s["width"], device="cuda")
    # given back: what a sequence holds past its positions, the last page first
    keep = torch.minimum((lens + page - 1) // page, s["held"].long())
    gone = (place >= keep[:, None]) & (place < s["held"][:, None])
    back = s["table"][gone].flip(0)
    s["free"][s["n_free"].long() + torch.arange(back.numel(), device="cuda")] = back
    s["n_free"] += back.numel()
    s["table"].masked_fill_(gone, -1)
    # taken: from the end of the list, sequence by sequence while there are enough
    need = torch.where(add > 0, ((lens + add + page - 1) // page - keep).clamp(min=0), 0)
    upto = need.cumsum(0)
    granted = (need == 0) | (upto <= s["n_free"].long())
    take = torch.where(granted, need, 0)
    taken = (place >= keep[:, None]) & (place < (keep + take)[:, None])
    at = s["n_free"].long() - 1 - (upto - need)[:, None] - (place - keep[:, None])
    s["table"].copy_(torch.where(taken, s["free"][at.clamp(0, s["pages"] - 1)], s["table"]))
    s["held"].copy_(keep + take)
    s["n_free"] -= take.sum().to(torch.int32)
    s["start"].copy_(torch.cat((torch.zeros_like(add[:1]), add.cumsum(0))))
    seq = torch.repeat_interleave(torch.arange(b, device="cuda"), add, output_size=s["n"])
    node = torch.arange(s["n"], device="cuda") - s["start"].long()[seq]
    slot = _slot(s["table"], page, seq, lens[seq] + node)
    s["slots"].copy_(torch.where(granted[seq], slot, -1))
    if c["tree"]:
        depth = (s["mask"][:, None] >> torch.arange(64, device="cuda") & 1).sum(-1) - 1
        s["pos"].copy_(lens[seq] + depth)
    else:
        s["pos"].copy_(lens[seq] + node)
    s["granted"].copy_(granted)
    return {k: s[k] for k in ("free", "n_free", "table", "held", "start", "slots", "pos", "granted")}


def _first(true):
    """The lowest place of each row that is true (the last one's after it where none is)."""
    at = torch.arange(true.shape[-1], device="cuda")
    return torch.where(true, at, true.shape[-1]).amin(-1)


def _plain_verify(c, s):
    n, b, m, vocab = s["n"], c["seqs"], c["tokens"], c["vocab"]
    start, lens, u, logits = s["start"].long(), s["len"].long(), s["u"].double(), s["logits"]
    news = start[1:] - start[:-1]
    seq = torch.repeat_interleave(torch.arange(b, device="cuda"), news, output_size=n)
    node = torch.arange(m, device="cuda")
    token = torch.where(node < news[:, None], start[:-1, None] + node, n)  # [seqs][m], n for none
    tokens = torch.cat((s["tokens"].long(), torch.full_like(start[:1], -1)))[token]
    # 64 bits: sums over a vocabulary decide between neighbouring tokens
    temp = s["temp"].double()[seq, None]
    top = logits.amax(-1, keepdim=True)
    likeliest = _first(logits == top)
    greedy = temp == 0
    w = torch.exp((logits.double() - top.double()) / torch.where(greedy, 1.0, temp))
    at = torch.arange(vocab, device="cuda")
    w = torch.where(greedy, (at == likeliest[:, None]).double(), w)
    cum = w.cumsum(-1)
    z = cum[:, -1:]
    picked = _first(cum > u[:, 1:] * z).clamp(max=vocab - 1)
    on_row = torch.cat((picked, torch.full_like(start[:1], -1)))[token]  # each node's row's choice
    if c["draft"]:
        follows = torch.cat((s["tokens"].long()[1:], torch.zeros_like(start[:1])))[:, None]  # the chain's next token
        rest = (w - z * s["draft"]).clamp(min=0)
        rest_cum = rest.cumsum(-1)
        other = _first(rest_cum > u[:, 1:] * rest_cum[:, -1:]).clamp(max=vocab - 1)
        other = torch.where(greedy[:, 0], likeliest, torch.where(rest_cum[:, -1] > 0, other, picked))
        passed = (u[:, :1] * s["draft"].gather(1, follows) * z < w.gather(1, follows))[:, 0]
        passed = torch.where(greedy[:, 0], likeliest == follows[:, 0], passed)
        passed = torch.cat((passed, torch.zeros_like(passed[:1])))[token]
        inside = node + 1 < news[:, None]
        on_path = torch.cat((torch.ones_like(passed[:, :1]), (passed & inside)[:, :-1].long().cumprod(-1).bool()), -1)
        on_row = torch.where(inside, torch.cat((other, torch.full_like(start[:1], -1)))[token], on_row)
    else:
        mask = s["mask"] if c["tree"] else (2 << torch.arange(n, device="cuda") - start[seq]) - 1
        bits = torch.cat((mask, torch.zeros_like(mask[:1])))[token][..., None] >> node & 1 == 1  # [seqs][node][ancestor]
        parent = torch.where(bits & (node < node[:, None]), node, -1).amax(-1)
        right = (tokens == on_row.gather(1, parent.clamp(min=0))) & (parent >= 0) & (token < n)
        same = (parent[:, :, None] == parent[:, None]) & (tokens[:, :, None] == tokens[:, None])
        right &= ~(same & (node < node[:, None])).any(-1)  # of children that say the same, the first
        right |= node == 0
        on_path = ~(bits & ~right[:, None]).any(-1) & right
    on_path &= token < n
    last = torch.where(on_path, node, -1).amax(-1)
    count = on_path.sum(-1)
    s["count"].copy_(count - 1)
    s["new_len"].copy_(lens + count)
    s["next"].copy_(on_row.gather(1, last[:, None])[:, 0])
    # the path's nodes in order, then what is said: its tokens after the first, and the next one
    path = torch.where(on_path, node, m).sort(-1).values
    said = torch.cat((tokens.gather(1, path.clamp(max=m - 1)), s["next"][:, None].long()), -1)[:, 1:]
    said = torch.where(node == count[:, None] - 1, s["next"][:, None].long(), said)
    said = torch.where(node < count[:, None], said, -1)
    flat = (token < n).view(-1)
    s["emit"].copy_(said.reshape(-1)[flat])
    moved = (path < m) & (path != node)
    place = lambda k: _slot(s["table"], s["page"], torch.arange(b, device="cuda")[:, None], lens[:, None] + k)  # noqa: E731
    s["src"].copy_(torch.where(moved, place(path.clamp(max=m - 1).minimum(news[:, None] - 1)), -1).reshape(-1)[flat])
    s["dst"].copy_(torch.where(moved, place(node.minimum(news[:, None] - 1)), -1).reshape(-1)[flat])
    return {k: s[k] for k in ("next", "count", "emit", "src", "dst", "new_len")}


def run(state):
    s, c = state, state["case"]
    if own:
        return _run_own(s, c)
    return {"chunk": _plain_chunk, "plan": _plain_plan, "verify": _plain_verify}[c["what"]](c, s)


# ---- the package's operators ----------------------------------------------------------------------------------------

_gemm = None  # the program's context on the GPU


def _own_parts(s, c):
    """The context, and the descriptors that a program keeps beside its buffers."""
    global _gemm
    from qwenny_amd import Gemm, KvCache, KvFmt, KvPool, TreeStep

    if _gemm is None:
        _gemm = Gemm.load(0)
    kept = s["kept"]
    if not kept:
        if c["what"] == "chunk":
            kept["kv"] = KvCache({"i8": KvFmt.I8, "e4m3": KvFmt.E4M3}[c["fmt"]], c["kv_heads"], c["dim"], c["page"], s["codes"],
                                 s["scales"])
        if c["what"] == "plan":
            kept["pool"] = KvPool(c["page"], s["free"], s["n_free"], s["table"], s["held"])
        else:
            kept["step"] = TreeStep(s["n"], s["start"], s["len"], s["table"], c["tokens"], s.get("mask"))
    return _gemm, kept


def _run_own(s, c):
    from qwenny_amd import kv_plan, kv_release

    gemm, kept = _own_parts(s, c)
    if c["what"] == "chunk":
        gemm.chunk_attn(None, s["q"], c["heads"], kept["kv"], kept["step"], s["out"], gate=s["gate"])
        return {"out": s["out"]}
    if c["what"] == "plan":
        kv_release(None, kept["pool"], s["len"])
        kv_plan(None, kept["pool"], s["len"], s["add"], s["n"], s["start"], s["slots"], s["pos"], s["granted"], mask=s["mask"])
        return {k: s[k] for k in ("free", "n_free", "table", "held", "start", "slots", "pos", "granted")}
    gemm.verify(None, s["logits"], c["vocab"], kept["step"], s["page"], s["tokens"], s["u"], s["next"], s["count"], s["emit"],
                temp=s["temp"], draft=s["draft"], src=s["src"], dst=s["dst"], new_len=s["new_len"])
    return {k: s[k] for k in ("next", "count", "emit", "src", "dst", "new_len")}


# ---- what a pass cannot do without, and the operators in 64 bits ----------------------------------------------------


def work(case):
    c = case
    if c["what"] == "verify":
        # each row's logits once, of the drafts' probabilities the row where a sequence ends
        n = sum(_drafted(c))
        return {"bytes": n * (c["vocab"] * 4 + 24) + (c["seqs"] * c["vocab"] * 4 if c["draft"] else 0),
                "flops": n * c["vocab"] * 20}
    lens, news = _requests(c)
    n = sum(news)
    if c["what"] == "plan":
        pages = sum(-(-(a + m) // c["page"]) - -(-a // c["page"]) for a, m in zip(lens, news)) + sum(_left_over(c))
        return {"bytes": 24 * c["seqs"] + n * (16 if c["tree"] else 8) + 8 * pages, "flops": n * 4 + c["seqs"] * 20}
    h, j, d = c["heads"], c["kv_heads"], c["dim"]
    seen = sum(m * a + m * (m + 1) // 2 for a, m in zip(lens, news))
    total = sum(a + m for a, m in zip(lens, news) if m)
    return {"bytes": total * j * (2 * d + 8) + n * h * d * 2 * (3 if c["gated"] else 2), "flops": 4 * h * d * seen}


def _exact_chunk(c, s):
    """Sequence by sequence, from the bytes."""
    lens, news = _requests(c)
    h, j, d, p = c["heads"], c["kv_heads"], c["dim"], c["page"]
    outs, row = [], 0
    for b, (a, m) in enumerate(zip(lens, news)):
        if not m:
            continue
        held = s["table"][b, : -(-(a + m) // p)].long()
        codes = s["codes"][held]
        if c["fmt"] == "i8":
            value = codes.to(torch.float64) - 128
        else:
            sign, e, f = codes >> 7, (codes >> 3 & 15).double(), (codes & 7).double()
            value = torch.where(e > 0, (1 + f / 8) * torch.exp2(e - 7), f * 2.0**-9) * (1 - 2 * sign.double())
        t = torch.arange(p, device="cuda")
        k = value[:, :, 0].view(len(held), j, p // 16, d // 64, 16, 64).transpose(3, 4).reshape(len(held), j, p, d)
        v = value[:, :, 1].view(len(held), j, p // 64, d, 64)[..., t[:64] % 16 // 4 * 16 + t[:64] // 16 * 4 + t[:64] % 4]
        v = v.transpose(3, 4).reshape(len(held), j, p, d)
        kv = torch.stack((k, v), 2) * s["scales"][held].double()[..., None]
        kv = kv.permute(1, 2, 0, 3, 4).reshape(j, 2, -1, d)[:, :, : a + m]
        qs = s["q"][row : row + m].double().view(m, j, h // j, d)
        late = torch.arange(a + m, device="cuda") > a + torch.arange(m, device="cuda")[:, None]
        heads = []
        for g in range(j):
            x = (qs[:, g].reshape(-1, d) @ kv[g, 0].T / math.sqrt(d)).view(m, h // j, -1)
            x = torch.softmax(x.masked_fill_(late[:, None], float("-inf")), -1)
            heads.append((x.view(-1, a + m) @ kv[g, 1]).view(m, h // j, d))
        outs.append(torch.cat(heads, 1))
        row += m
    out = torch.cat(outs)
    return {"out": out / (1 + torch.exp(-s["gate"].double())) if c["gated"] else out}


def _exact_plan(c, s):
    """As a list of pages that requests push to and pop from."""
    page = c["page"]
    host = {k: s[k].tolist() for k in ("free", "n_free", "table", "held", "len", "add")}
    free, count, table, held = host["free"], host["n_free"][0], host["table"], host["held"]
    stack, rest = free[:count], free[count:]
    for b in reversed(range(c["seqs"])):
        while held[b] > -(-host["len"][b] // page):
            held[b] -= 1
            stack.append(table[b][held[b]])
            table[b][held[b]] = -1
    free = stack + free[len(stack):]
    granted, asked, had = [], 0, len(stack)
    start, slots, pos = [0], [], []
    masks = s["mask"].tolist() if c["tree"] else None
    for b, (a, m) in enumerate(zip(host["len"], host["add"])):
        need = max(0, -(-(a + m) // page) - held[b]) if m else 0
        asked += need
        granted.append(int(need == 0 or asked <= had))
        if granted[-1]:
            for _ in range(need):
                table[b][held[b]] = stack.pop()
                held[b] += 1
        for i in range(m):
            t = a + i
            slots.append(table[b][t // page] * page + t % page if granted[-1] else -1)
            pos.append(a + (bin(masks[len(pos)] & (1 << 64) - 1).count("1") - 1 if c["tree"] else i))
        start.append(start[-1] + m)
    return {"free": _dev(free), "n_free": _dev([len(stack)]), "table": _dev(table), "held": _dev(held), "start": _dev(start),
            "slots": _dev(slots), "pos": _dev(pos), "granted": _dev(granted)}


def _exact_verify(c, s):
    """Sequence by sequence, walking from token to token."""
    host = {k: s[k].tolist() for k in ("start", "len", "table", "tokens", "temp", "u")}
    masks = s["mask"].tolist() if c["tree"] else None
    got = {k: [] for k in ("next", "count", "emit", "src", "dst", "new_len")}

    def chances(row, temp):
        x = s["logits"][row].double()
        if temp == 0:
            return torch.zeros_like(x).index_fill_(0, torch.nonzero(x == x.max())[0], 1.0)
        return torch.softmax(x / temp, -1)

    def choose(p, u):
        cum = torch.cumsum(p, 0)
        return min(int(torch.searchsorted(cum, u * cum[-1], right=True)), len(p) - 1)

    for b, temp in enumerate(host["temp"]):
        a, m = host["start"][b], host["start"][b + 1] - host["start"][b]
        said = host["tokens"][a : a + m]
        parents = [-1] + [((masks[a + i] & (1 << 64) - 1 ^ 1 << i).bit_length() - 1) if c["tree"] else i - 1 for i in range(1, m)]
        path, nxt = [0], None
        while nxt is None:
            i = path[-1]
            p, (u0, u1) = chances(a + i, temp), host["u"][a + i]
            if c["draft"] and i + 1 < m:
                t, q = said[i + 1], s["draft"][a + i].double()
                if temp == 0:
                    ok = bool(p[t] == 1)
                else:
                    ok = u0 * float(q[t]) < float(p[t])
                if ok:
                    path.append(i + 1)
                elif temp == 0:
                    nxt = int(p.argmax())
                else:
                    rest = (p - q).clamp(min=0)
                    nxt = choose(rest if float(rest.sum()) > 0 else p, u1)
                continue
            y = choose(p, u1)
            child = [k for k in range(i + 1, m) if parents[k] == i and said[k] == y and not c["draft"]]
            if child:
                path.append(child[0])
            else:
                nxt = y
        place = lambda k: host["table"][b][(host["len"][b] + k) // s["page"]] * s["page"] + (host["len"][b] + k) % s["page"]  # noqa: E731, B023
        got["next"].append(nxt)
        got["count"].append(len(path) - 1)
        got["new_len"].append(host["len"][b] + len(path))
        got["emit"] += [said[k] for k in path[1:]] + [nxt] + [-1] * (m - len(path))
        got["src"] += [place(k) if k != i else -1 for i, k in enumerate(path)] + [-1] * (m - len(path))
        got["dst"] += [place(i) if k != i else -1 for i, k in enumerate(path)] + [-1] * (m - len(path))
    return {k: _dev(v) for k, v in got.items()}


def exact(case, seed):
    c, s = case, prepare(case, seed)
    return {"chunk": _exact_chunk, "plan": _exact_plan, "verify": _exact_verify}[c["what"]](c, s)
