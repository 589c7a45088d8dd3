"""The attention of a decode step over a quantised, paged KV cache: what is measured of it.

Four kinds of work. `prep`: the in-projection's split-K partials summed, queries and keys normed per head and rotated to
their positions, into dense bf16 q, gate, k, v. `cache`: keys and values quantised into cache slots, and the same slots
read back. `attn`: drafted tokens (a chain, or a tree with a mask of ancestors) and single tokens attending over the
cache. `step`: what an engine runs between the in-projection and the out-projection of one layer: prep straight into
the cache, attention, and the accepted path's slots moved together, read back.

The cache is two buffers, codes u8 [pages][kv heads][2][page * dim] and scales f32 [pages][kv heads][2][page], keys then
values. Token t of a page, dimension d, lies in the keys' block at
    (t / 16) * 16 dim + (d / 64) * 1024 + (t % 16) * 64 + d % 64
and in the values' at
    (t / 64) * 64 dim + d * 64 + (t % 16 / 4) * 16 + (t % 64 / 16) * 4 + t % 4.
i8 codes are q + 128 with scale max|v| / 127, e4m3 codes are the type's bytes with scale max|v| / 448; a slot is its page
times the page's length plus its place in it."""

import math
import random

import torch

own = False

EPS = 1e-6
THETA = 1e7
TOP = {"i8": 127.0, "e4m3": 448.0}

# attention of the two model sizes that the package is measured on: gated queries, a quarter of each head rotated
SIZE_4B = {"heads": 16, "kv_heads": 4, "dim": 256, "rot": 64, "gated": True}
SIZE_27B = {"heads": 24, "kv_heads": 4, "dim": 256, "rot": 64, "gated": True}
# a grouped-query layer without gates, whole heads rotated
SIZE_GQA = {"heads": 32, "kv_heads": 8, "dim": 128, "rot": 128, "gated": False}


def _attn(name, fmt, size, seqs, lo, hi, tokens, tree, page=256, what="attn"):
    return {"name": name, "what": what, "fmt": fmt, **size, "page": page, "seqs": seqs, "len_lo": lo, "len_hi": hi,
            "tokens": tokens, "tree": tree}


def listed():
    return [
        # decode, one token: the in-projection's eight partials of a small model
        {"name": "prep_4b_1", "what": "prep", **SIZE_4B, "n": 1, "splits": 8},
        # the largest prompt chunk: one partial, dense queries and keys for a prompt's attention
        {"name": "prep_27b_2048", "what": "prep", **SIZE_27B, "n": 2048, "splits": 1},
        # a few tokens written and handed on
        {"name": "cache_e4m3_9", "what": "cache", "fmt": "e4m3", "kv_heads": 8, "dim": 128, "page": 64, "n": 9},
        # a prompt chunk written and read back (a session that is saved, a prefix that is shared)
        {"name": "cache_i8_2048", "what": "cache", "fmt": "i8", "kv_heads": 4, "dim": 256, "page": 256, "n": 2048},
        # the smallest call: one token early in a conversation
        _attn("attn_4b_1_len77", "i8", SIZE_4B, 1, 77, 77, 1, False),
        # plain decode
        _attn("attn_27b_1_len4k", "i8", SIZE_27B, 1, 4099, 4099, 1, False),
        # four drafted tokens after the accepted one, a long context
        _attn("attn_27b_5_len32k", "i8", SIZE_27B, 1, 32700, 32700, 5, False),
        # the longest context
        _attn("attn_27b_1_len128k", "e4m3", SIZE_27B, 1, 131000, 131000, 1, False),
        # a batch of sequences of very different lengths
        _attn("attn_27b_batch32", "i8", SIZE_27B, 32, 100, 8000, 1, False),
        # the largest tree
        _attn("attn_27b_tree64_len8k", "i8", SIZE_27B, 1, 8150, 8150, 64, True),
        # one layer of a verification step
        _attn("step_27b_5_len4k", "i8", SIZE_27B, 1, 4090, 4090, 5, True, what="step"),
        # one layer of a batch that verifies small trees
        _attn("step_gqa_tree8_batch8", "e4m3", SIZE_GQA, 8, 500, 4000, 8, True, page=64, what="step"),
    ]


def _log(rng, lo, hi):
    return int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))


def draw(rng):
    dim = rng.choice((64, 128, 256))
    kv_heads = rng.choice((1, 2, 4, 8))
    size = {"heads": kv_heads * rng.choice((1, 2, 3, 4, 5, 6, 8)), "kv_heads": kv_heads, "dim": dim,
            "rot": rng.choice((dim // 4, dim // 2, dim)), "gated": rng.random() < 0.5}
    fmt, page = rng.choice(("i8", "e4m3")), rng.choice((64, 128, 256))
    what = rng.choices(("prep", "cache", "attn", "step"), (2, 2, 5, 2))[0]
    if what == "prep":
        n = _log(rng, 1, 2000)
        return {"what": what, **size, "n": n, "splits": rng.choice((1, 2, 3, 5, 10)) if n <= 48 else 1}
    if what == "cache":
        return {"what": what, "fmt": fmt, "kv_heads": kv_heads, "dim": dim, "page": page, "n": _log(rng, 1, 4000)}
    tokens = rng.choice((1, 1, 2, 3, 5, 8, 13, 31, 64))
    seqs = _log(rng, 1, 40) if tokens < 31 else _log(rng, 1, 4)
    hi = _log(rng, 40, min(130000, 4 * 256 * 130000 // (kv_heads * dim * seqs), 600000 // (tokens * seqs)))
    lo = max(1, int(hi * rng.uniform(0.02, 1.0)))
    return {"what": what, "fmt": fmt, **size, "page": page, "seqs": seqs, "len_lo": lo, "len_hi": hi, "tokens": tokens,
            "tree": tokens > 1 and rng.random() < 0.6}


# ---- inputs ---------------------------------------------------------------------------------------------------------


def _gen(seed, name):
    g = torch.Generator(device="cuda")
    g.manual_seed((seed * 1_000_003 + sum((i + 1) * ord(c) for i, c in enumerate(name))) & 0x7FFFFFFFFFFF)
    return g


def _dev(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


def _rng(c):
    return random.Random("%s %s %s %s" % (c["seqs"], c["len_lo"], c["len_hi"], c["tokens"]))


def _plan(c):
    """(cached tokens, new tokens) of each sequence: the same for every seed. Of four sequences and more, one has
    nothing new in this step and one nothing cached yet."""
    rng = _rng(c)
    lens = [max(c["len_lo"], min(c["len_hi"], _log(rng, c["len_lo"], c["len_hi"]))) for _ in range(c["seqs"])]
    news = [rng.randint(1, c["tokens"]) for _ in range(c["seqs"])]
    lens[0], news[0] = c["len_hi"], c["tokens"]
    if c["seqs"] >= 4:
        news[1], lens[2] = 0, 0
    return lens, news


def _ancestors(rng, n, tree):
    """Masks of the nodes each node sees (itself and its ancestors) and the nodes' depths; a chain, or parents at random."""
    masks, depths = [], []
    for i in range(n):
        parent = i - 1 if not tree else rng.randint(-1, i - 1)
        masks.append((masks[parent] if parent >= 0 else 0) | 1 << i)
        depths.append(depths[parent] + 1 if parent >= 0 else 0)
    return masks, depths


def _signed(u):
    return u - (1 << 64) if u >> 63 else u


def _cache(c, g, pages):
    """A filled cache: bell-shaped codes, a scale of its own for each vector."""
    shape = (pages, c["kv_heads"], 2, c["page"] * c["dim"])
    values = torch.randn(shape, generator=g, device="cuda", dtype=torch.float16 if math.prod(shape) > 1 << 26 else torch.float32)
    if c["fmt"] == "i8":
        codes = ((values * 40).round_().clamp_(-127, 127) + 128).to(torch.uint8)
        size = 0.025
    else:
        codes = (values * 100).clamp_(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
        size = 0.01
    scales = torch.rand(shape[:3] + (c["page"],), generator=g, device="cuda") * size + 0.5 * size
    return codes, scales


def _prep_inputs(c, g, n, splits, positions):
    rows = (c["heads"] * (2 if c["gated"] else 1) + 2 * c["kv_heads"]) * c["dim"]
    s = {"x": torch.randn((splits, n, rows), generator=g, device="cuda") * 1.5,
         "q_w": torch.rand(c["dim"], generator=g, device="cuda") + 0.5,
         "k_w": torch.rand(c["dim"], generator=g, device="cuda") + 0.5,
         "inv_freq": (THETA ** (-torch.arange(0, c["rot"], 2, device="cuda", dtype=torch.float64) / c["rot"])).float(),
         "pos": positions, "n": n, "splits": splits}
    s["q"] = torch.empty((n, c["heads"], c["dim"]), dtype=torch.bfloat16, device="cuda")
    s["gate"] = torch.empty_like(s["q"]) if c["gated"] else None
    return s


def prepare(case, seed):
    c = case
    g = _gen(seed, c["what"])
    s = {"case": c, "kept": {}}
    if c["what"] in ("prep", "cache"):
        n = c["n"]
        kv_shape = (n, c["kv_heads"], c["dim"])
        if c["what"] == "prep":
            first = random.Random(seed).randint(0, 250_000)  # a chunk of a long prompt
            s |= _prep_inputs(c, g, n, c["splits"], torch.arange(first, first + n, dtype=torch.int32, device="cuda"))
            s["k"], s["v"] = (torch.empty(kv_shape, dtype=torch.bfloat16, device="cuda") for _ in range(2))
            return s
        s["k"], s["v"] = (torch.randn(kv_shape, generator=g, device="cuda").to(torch.bfloat16) for _ in range(2))
        first = random.Random(seed).randint(0, 3 * c["page"])  # in the middle of a sequence whose pages lie anywhere
        pages = (first + n) // c["page"] + 3
        s["codes"], s["scales"] = _cache(c, g, pages)
        table = torch.randperm(pages, generator=g, device="cuda")
        at = torch.arange(first, first + n, device="cuda")
        s["slots"] = (table[at // c["page"]] * c["page"] + at % c["page"]).to(torch.int32)
        s["k_back"], s["v_back"] = torch.empty_like(s["k"]), torch.empty_like(s["v"])
        return s
    lens, news = _plan(c)
    rng = random.Random(seed)
    held = [-(-(a + b) // c["page"]) for a, b in zip(lens, news)]
    pages = sum(held) + 2
    order = list(range(pages))
    rng.shuffle(order)
    width = max(max(held), 1)
    table = [[order.pop() for _ in range(h)] for h in held]
    s["codes"], s["scales"] = _cache(c, g, pages)
    used = _dev([p for row in table for p in row], torch.int64)
    place = _dev([k for h in held for k in range(h)], torch.int64)
    total = _dev([a + b for a, b, h in zip(lens, news, held) for _ in range(h)], torch.int64)
    written = torch.zeros((pages, c["page"]), dtype=torch.bool, device="cuda")
    if len(used):
        written[used] = place[:, None] * c["page"] + torch.arange(c["page"], device="cuda") < total[:, None]
    # what no sequence has written is whatever the memory held
    s["scales"] = torch.where(written[:, None, None, :], s["scales"], float("nan"))
    n = sum(news)
    rng = _rng(c)  # trees and accepted paths, too, are the same for every seed
    masks, depths, start = [], [], [0]
    path_src, path_dst, path_start = [], [], [0]
    slot = lambda b, i: table[b][(lens[b] + i) // c["page"]] * c["page"] + (lens[b] + i) % c["page"]  # noqa: E731
    for b, m in enumerate(news):
        k, d = _ancestors(rng, m, c["tree"])
        masks += [_signed(v) for v in k]
        depths += [lens[b] + v for v in d]
        start.append(start[-1] + m)
        last = rng.randint(0, m - 1) if m else 0
        path = [i for i in range(m) if k[last] >> i & 1]
        path_src += [slot(b, i) for i in path]
        path_dst += [slot(b, i) for i in range(len(path))]
        path_start.append(len(path_src))
    s |= {"start": _dev(start), "len": _dev(lens), "table": _dev([row + [-1] * (width - len(row)) for row in table]),
          "mask": _dev(masks, torch.int64) if c["tree"] else None, "n": n, "width": width}
    if c["what"] == "attn":
        strength = torch.rand((n, c["heads"], 1), generator=g, device="cuda") * 3 + 0.3  # flat and peaked heads
        s["q"] = (torch.randn((n, c["heads"], c["dim"]), generator=g, device="cuda") * strength).to(torch.bfloat16)
        s["gate"] = torch.randn(s["q"].shape, generator=g, device="cuda").to(torch.bfloat16) if c["gated"] else None
    else:
        splits = 4 if n <= 48 else 1
        s |= _prep_inputs(c, g, n, splits, _dev(depths))
        s["slots"] = _dev([slot(b, i) for b in range(c["seqs"]) for i in range(news[b])])
        s |= {"path_src": _dev(path_src), "path_dst": _dev(path_dst), "path_start": _dev(path_start)}
        s["k_back"], s["v_back"] = (torch.empty((len(path_dst), c["kv_heads"], c["dim"]), dtype=torch.bfloat16, device="cuda")
                                    for _ in range(2))
    s["out"] = torch.empty_like(s["q"])
    return s


# ---- the plain form -------------------------------------------------------------------------------------------------


def _places(c, slots):
    """Where the codes of keys and values of `slots` lie in the flat buffer, [n][kv heads][2][dim], and their scales'."""
    slots = slots.long()
    page, t = slots // c["page"], slots % c["page"]
    d = torch.arange(c["dim"], device=slots.device)
    t1 = t[:, None]
    k = t1 // 16 * (16 * c["dim"]) + d // 64 * 1024 + t1 % 16 * 64 + d % 64
    v = t1 // 64 * (64 * c["dim"]) + d * 64 + t1 % 16 // 4 * 16 + t1 % 64 // 16 * 4 + t1 % 4
    block = (page[:, None] * c["kv_heads"] + torch.arange(c["kv_heads"], device=slots.device))[:, :, None] * 2
    block = block + torch.arange(2, device=slots.device)
    codes = block[..., None] * (c["page"] * c["dim"]) + torch.stack((k, v), 1)[:, None]
    return codes, block * c["page"] + t[:, None, None]


def _values(c, codes):
    return codes.float() - 128 if c["fmt"] == "i8" else codes.view(torch.float8_e4m3fn).float()


def _write(c, s, slots, kv):
    """kv f32 [n][kv heads][2][dim] quantised into the cache."""
    codes_at, scales_at = _places(c, slots)
    scale = (kv.abs().amax(-1).double() / TOP[c["fmt"]]).float()  # divided in 64 bits: values next to a code's border
    scaled = torch.where(scale[..., None] > 0, kv.double() / scale[..., None].double(), 0.0)
    if c["fmt"] == "i8":
        codes = (scaled.round().clamp(-127, 127) + 128).to(torch.uint8)
    else:
        unit = torch.ldexp(torch.ones_like(scaled), torch.frexp(scaled).exponent.clamp(min=-5) - 4)  # 3 bits behind the first
        codes = ((scaled / unit).round() * unit).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
    s["codes"].view(-1)[codes_at] = codes
    s["scales"].view(-1)[scales_at] = scale


def _read(c, s, slots):
    codes_at, scales_at = _places(c, slots)
    kv = _values(c, s["codes"].view(-1)[codes_at]) * s["scales"].view(-1)[scales_at][..., None]
    return kv.to(torch.bfloat16)


def _norm_rotate(x, w, c, cos, sin):
    x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w
    a, b, rest = x.split((c["rot"] // 2, c["rot"] // 2, c["dim"] - c["rot"]), -1)
    return torch.cat((a * cos - b * sin, b * cos + a * sin, rest), -1)


def _prep(c, s):
    """f32 q, gate, k, v of the in-projection's partials."""
    n, h, j, d = s["n"], c["heads"], c["kv_heads"], c["dim"]
    x = s["x"].sum(0)
    per = 2 * d if c["gated"] else d
    q, k, v = x.split((h * per, j * d, j * d), -1)
    q = q.reshape(n, h, per)
    angle = s["pos"].double()[:, None, None] * s["inv_freq"].double()
    cos, sin = angle.cos().float(), angle.sin().float()
    gate = q[..., d:] if c["gated"] else None
    return (_norm_rotate(q[..., :d], s["q_w"], c, cos, sin), gate, _norm_rotate(k.reshape(n, j, d), s["k_w"], c, cos, sin),
            v.reshape(n, j, d))


def _history(c, s):
    """The sequences' keys and values from the cache, f32 [seqs][kv heads][positions][dim] each; pages that a sequence
    has not are taken from page 0."""
    b, w, j, d, p = c["seqs"], s["width"], c["kv_heads"], c["dim"], c["page"]
    table = s["table"].long().clamp(min=0)
    codes, scales = s["codes"][table], s["scales"][table]
    k = _values(c, codes[:, :, :, 0]).view(b, w, j, p // 16, d // 64, 16, 64).permute(0, 2, 1, 3, 5, 4, 6)
    v = _values(c, codes[:, :, :, 1]).view(b, w, j, p // 64, d, 4, 4, 4).permute(0, 2, 1, 3, 6, 5, 7, 4)
    at = scales.permute(3, 0, 2, 1, 4).reshape(2, b, j, w * p, 1)
    return k.reshape(b, j, w * p, d) * at[0], v.reshape(b, j, w * p, d) * at[1]


def _attend(c, s, q, gate):
    """q, gate f32 [n][heads][dim] -> the gated attention, f32."""
    b, j, d, m = c["seqs"], c["kv_heads"], c["dim"], c["tokens"]
    group = c["heads"] // j
    start, lens = s["start"].long(), s["len"].long()
    node = torch.arange(m, device=q.device)
    news = start[1:] - start[:-1]
    token = torch.where(node < news[:, None], start[:-1, None] + node, s["n"])  # [seqs][m], padded with a token of zeros
    padded = torch.cat((q, torch.zeros_like(q[:1])))[token].view(b, m, j, group, d).permute(0, 2, 1, 3, 4)
    k, v = _history(c, s)
    at = torch.arange(k.shape[2], device=q.device)
    own_node = at - lens[:, None]  # [seqs][positions]: which of the step's nodes lies there
    if s["mask"] is None:
        sees = own_node[:, None] <= node[:, None]
    else:
        bits = torch.cat((s["mask"], torch.zeros_like(s["mask"][:1])))[token]
        sees = (own_node[:, None] < 0) | (bits[..., None] >> own_node[:, None].clamp(0, 63) & 1 == 1)
    held = (own_node < news[:, None])[:, None, :, None]
    k, v = torch.where(held, k, 0.0), torch.where(held, v, 0.0)
    sees = (sees & (own_node < news[:, None])[:, None])[:, None, :, None]  # [seqs][1][m][1][positions]
    scores = torch.matmul(padded.reshape(b, j, m * group, d), k.transpose(-1, -2)).view(b, j, m, group, -1) * d**-0.5
    scores = torch.where(sees, scores, float("-inf"))
    p = torch.exp(scores - scores.amax(-1, keepdim=True).clamp(min=-1e30))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total > 0, total, 1.0)
    o = torch.matmul(p.view(b, j, m * group, -1), v).view(b, j, m, group, d).permute(0, 2, 1, 3, 4).reshape(b * m, -1, d)
    o = o[(node < news[:, None]).view(-1)]
    return o * torch.sigmoid(gate) if gate is not None else o


def _bf(x):
    return None if x is None else x.to(torch.bfloat16)


def _move(c, s):
    """The accepted path's codes and scales put together: all read, then written."""
    from_codes, from_scales = _places(c, s["path_src"])
    to_codes, to_scales = _places(c, s["path_dst"])
    codes, scales = s["codes"].view(-1)[from_codes], s["scales"].view(-1)[from_scales]
    s["codes"].view(-1)[to_codes] = codes
    s["scales"].view(-1)[to_scales] = scales


def _outputs(s, **more):
    return {k: v for k, v in more.items() if v is not None}


def run(state):
    s, c = state, state["case"]
    if own:
        return _run_own(s, c)
    if c["what"] == "prep":
        q, gate, k, v = _prep(c, s)
        return _outputs(s, q=_bf(q), gate=_bf(gate), k=_bf(k), v=_bf(v))
    if c["what"] == "cache":
        _write(c, s, s["slots"], torch.stack((s["k"], s["v"]), 2).float())
        back = _read(c, s, s["slots"])
        return _outputs(s, k=back[:, :, 0], v=back[:, :, 1])
    if c["what"] == "attn":
        return _outputs(s, out=_bf(_attend(c, s, s["q"].float(), None if s["gate"] is None else s["gate"].float())))
    q, gate, k, v = _prep(c, s)
    _write(c, s, s["slots"], torch.stack((k, v), 2))
    q, gate = _bf(q), _bf(gate)
    out = _bf(_attend(c, s, q.float(), None if gate is None else gate.float()))
    _move(c, s)
    back = _read(c, s, s["path_dst"])
    return _outputs(s, q=q, gate=gate, out=out, k=back[:, :, 0], v=back[:, :, 1])


# ---- the package's operators ----------------------------------------------------------------------------------------

_gemm = None  # the program's context on the GPU


def _own_parts(s, c):
    """The context, and the descriptors that a program keeps beside its buffers."""
    global _gemm
    from qwenny_amd import AttnRows, Gemm, KvCache, KvFmt, TreeStep

    if _gemm is None:
        _gemm = Gemm.load(0)
    kept = s["kept"]
    if not kept:
        if "codes" in s:
            kept["kv"] = KvCache({"i8": KvFmt.I8, "e4m3": KvFmt.E4M3}[c["fmt"]], c["kv_heads"], c["dim"], c["page"], s["codes"],
                                 s["scales"])
        if "table" in s:
            kept["step"] = TreeStep(s["n"], s["start"], s["len"], s["table"], c["tokens"], s["mask"])
        if "x" in s:
            kept["rows"] = AttnRows(c["heads"], c["kv_heads"], c["dim"], c["rot"], c["gated"])
    return _gemm, kept


def _run_own(s, c):
    from qwenny_amd import attn_prep, kv_move, kv_read, kv_write

    gemm, kept = _own_parts(s, c)
    if c["what"] == "prep":
        attn_prep(None, s["x"], s["splits"], s["n"], kept["rows"], s["q_w"], s["k_w"], s["inv_freq"], s["pos"], s["q"], s["gate"],
                  k=s["k"], v=s["v"], eps=EPS)
        return _outputs(s, q=s["q"], gate=s["gate"], k=s["k"], v=s["v"])
    if c["what"] == "cache":
        kv_write(None, kept["kv"], s["k"], s["v"], s["slots"], c["n"])
        kv_read(None, kept["kv"], s["slots"], c["n"], s["k_back"], s["v_back"])
        return _outputs(s, k=s["k_back"], v=s["v_back"])
    if c["what"] == "attn":
        gemm.tree_attn(None, s["q"], c["heads"], kept["kv"], kept["step"], s["out"], gate=s["gate"])
        return _outputs(s, out=s["out"])
    attn_prep(None, s["x"], s["splits"], s["n"], kept["rows"], s["q_w"], s["k_w"], s["inv_freq"], s["pos"], s["q"], s["gate"],
              kv=kept["kv"], slots=s["slots"], eps=EPS)
    gemm.tree_attn(None, s["q"], c["heads"], kept["kv"], kept["step"], s["out"], gate=s["gate"])
    kv_move(None, kept["kv"], s["path_src"], s["path_dst"], s["path_start"], c["seqs"])
    kv_read(None, kept["kv"], s["path_dst"], s["path_dst"].numel(), s["k_back"], s["v_back"])
    return _outputs(s, q=s["q"], gate=s["gate"], out=s["out"], k=s["k_back"], v=s["v_back"])


# ---- what a pass cannot do without, and the operators in 64 bits ----------------------------------------------------


def work(case):
    c = case
    j, d = c["kv_heads"], c["dim"]
    if c["what"] == "cache":
        n = c["n"]
        return {"bytes": n * (2 * j * d * 2 + 2 * j * (d + 4) + 2 * j * d * 2 + 4), "flops": n * 2 * j * d * 5}
    h = c["heads"]
    qo = h * d * 2 * (2 if c["gated"] else 1)  # bf16 q and gate of a token
    rows = (h * (2 if c["gated"] else 1) + 2 * j) * d
    if c["what"] == "prep":
        n = c["n"]
        return {"bytes": n * (c["splits"] * rows * 4 + qo + 2 * j * d * 2 + 4) + d * 8,
                "flops": n * (c["splits"] * rows + (h + j) * d * 8)}
    lens, news = _plan(c)
    n = sum(news)
    seen = sum(m * a + (m * (m + 1) // 2 if not c["tree"] else m) for a, m in zip(lens, news))
    total = sum(a + m for a, m in zip(lens, news) if m)
    w = {"bytes": total * j * (2 * d + 8) + n * (qo + h * d * 2), "flops": 4 * h * d * seen}
    if c["what"] == "step":
        splits = 4 if n <= 48 else 1
        w["bytes"] += n * (splits * rows * 4 + 2 * j * (d + 4)) + len(news) * 2 * j * d * 2
        w["flops"] += n * (splits * rows + (h + j) * d * 8)
    return w


def _exact_write(c, kv, scales, values, slots):
    """kv f64 [n][kv heads][2][dim] as the cache holds it: scales in f32, codes rounded to the nearest; `values` and
    `scales` are by slot."""
    scale = (kv.abs().amax(-1) / TOP[c["fmt"]]).float().double()
    u = torch.where(scale[..., None] > 0, kv / scale[..., None], 0.0)
    if c["fmt"] == "i8":
        u = u.round().clamp(-127, 127)
    else:
        step = torch.exp2(torch.floor(torch.log2(u.abs().clamp(min=2.0**-6))) - 3)
        u = ((u / step).round() * step).clamp(-448, 448)
    values[slots], scales[slots] = u, scale


def _exact_cache(c, codes, scales, slots):
    """(values f64, scales f64) of `slots`, from the bytes: [n][kv heads][2][dim] and [n][kv heads][2]."""
    p, d = c["page"], c["dim"]
    pages = codes.shape[0]
    if c["fmt"] == "i8":
        u = codes.to(torch.float64) - 128
    else:
        sign, e, f = codes >> 7, (codes >> 3 & 15).double(), (codes & 7).double()
        u = torch.where(e > 0, (1 + f / 8) * torch.exp2(e - 7), f * 2.0**-9) * (1 - 2 * sign.double())
        u = torch.where((codes & 127) == 127, float("nan"), u)
    t = torch.arange(p, device=codes.device)
    k = u[:, :, 0].view(pages, -1, p // 16, d // 64, 16, 64).transpose(3, 4).reshape(pages, -1, p, d)
    v = u[:, :, 1].view(pages, -1, p // 64, d, 64)[..., t[:64] % 16 // 4 * 16 + t[:64] // 16 * 4 + t[:64] % 4]
    v = v.transpose(3, 4).reshape(pages, -1, p, d)
    both = torch.stack((k, v), 3).transpose(1, 2).reshape(pages * p, -1, 2, d)
    sc = scales.double().permute(0, 3, 1, 2).reshape(pages * p, -1, 2)
    return both[slots], sc[slots]


def _exact_heads(x, w, pos, inv_freq, rot):
    y = x / (x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt() * w.double()
    z = torch.view_as_complex(torch.stack((y[..., : rot // 2], y[..., rot // 2 : rot]), -1).contiguous())
    turn = pos.double()[:, None] * inv_freq.double()
    z = z * torch.polar(torch.ones_like(turn), turn)[:, None]
    return torch.cat((z.real, z.imag, y[..., rot:]), -1)


def _exact_prep(c, s):
    n, h, j, d = s["n"], c["heads"], c["kv_heads"], c["dim"]
    x = s["x"].double().sum(0).view(n, -1, d)
    nq = h * 2 if c["gated"] else h
    q = x[:, :nq:2] if c["gated"] else x[:, :nq]
    gate = x[:, 1:nq:2] if c["gated"] else None
    q = _exact_heads(q, s["q_w"], s["pos"], s["inv_freq"], c["rot"])
    k = _exact_heads(x[:, nq : nq + j], s["k_w"], s["pos"], s["inv_freq"], c["rot"])
    return q, gate, k, x[:, nq + j :]


def _some(**more):
    return {k: v for k, v in more.items() if v is not None}


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["what"] == "prep":
        q, gate, k, v = _exact_prep(c, s)
        return _some(q=q, gate=gate, k=k, v=v)
    if c["what"] == "cache":
        kv = torch.stack((s["k"], s["v"]), 2).double()
        values, scales = torch.empty_like(kv), kv.new_empty(kv.shape[:3])
        _exact_write(c, kv, scales, values, torch.arange(c["n"], device="cuda"))
        back = values * scales[..., None]
        return _some(k=back[:, :, 0], v=back[:, :, 1])
    lens, news = _plan(c)
    h, j, d = c["heads"], c["kv_heads"], c["dim"]
    q, gate = s["q"], s["gate"]
    fresh = None
    if c["what"] == "step":
        q, gate, k, v = _exact_prep(c, s)
        kv = torch.stack((k, v), 2)
        values, scales = torch.empty_like(kv), kv.new_empty(kv.shape[:3])
        _exact_write(c, kv, scales, values, torch.arange(s["n"], device="cuda"))
        fresh = values * scales[..., None]
    outs, moved, row = [], [], 0
    for b, (a, m) in enumerate(zip(lens, news)):
        if not m:
            continue
        at = torch.arange(a + m, device="cuda")
        slots = s["table"][b].long()[at // c["page"]] * c["page"] + at % c["page"]
        held, place = torch.unique(s["table"][b, : -(-(a + m) // c["page"])].long(), return_inverse=True)
        values, scales = _exact_cache(c, s["codes"][held], s["scales"][held],
                                      place[at // c["page"]] * c["page"] + slots % c["page"])
        kv = values * scales[..., None]
        if fresh is not None:
            kv[a:] = fresh[row : row + m]
            mine = s["slots"][row : row + m].tolist()
            moved += [row + mine.index(v) for v in s["path_src"][s["path_start"][b] : s["path_start"][b + 1]].tolist()]
        qs = q[row : row + m].double().view(m, j, h // j, d).permute(1, 0, 2, 3).reshape(j, -1, d)
        scores = (qs @ kv[:, :, 0].permute(1, 2, 0)).view(j, m, h // j, -1) / math.sqrt(d)
        node = torch.arange(m, device="cuda")
        bits = s["mask"][row : row + m] if c["tree"] else None
        sees = (bits[:, None] >> node & 1).bool() if c["tree"] else node[None] <= node[:, None]
        scores[..., a:].masked_fill_(~sees[None, :, None], float("-inf"))
        o = torch.softmax(scores, -1).view(j, -1, a + m) @ kv[:, :, 1].transpose(0, 1)
        outs.append(o.view(j, m, h // j, d).permute(1, 0, 2, 3).reshape(m, h, d))
        row += m
    out = torch.cat(outs)
    out = out if gate is None else out / (1 + torch.exp(-gate.double()))
    if c["what"] == "attn":
        return _some(out=out)
    back = fresh[moved]
    return _some(q=q, gate=gate, out=out, k=back[:, :, 0], v=back[:, :, 1])
