"""A server's steps on the GPU: pages planned from the requests' lengths, prompts in chunks, trees of drafts verified and their paths
moved together, pages given back, requests that wait for pages and one that takes an ended one's place. The attention is held against
a plain form in 64 bits over the requests' texts, the cache bit for bit against one that was written in order."""

import numpy as np
import pytest
import torch

from qwenny_amd import AttnRows, Graph, KvCache, KvFmt, KvPool, TreeStep, attn_prep, kv_move, kv_plan, kv_release
from tests.test_chunk_attn_gpu import Chunk
from tests.test_kv_attn_gpu import Host, Step, _dev, _f64, new_cache
from tests.test_verify_gpu import _chances, _choose

pytestmark = pytest.mark.gpu

HEADS, KV_HEADS, DIM, ROT, PAGE, VOCAB, N_SEQ, WIDTH = 6, 2, 128, 64, 64, 301, 3, 6
MASKS, PARENTS, DEPTHS = [0b1, 0b11, 0b111, 0b1001, 0b11001], [-1, 0, 1, 0, 3], [0, 1, 2, 1, 2]
I32, BF16 = torch.int32, torch.bfloat16


class Server:
    """In place of a model: tables of a token's in-projection and of the logits after it."""

    def __init__(self, gemm, fmt, pages):
        g = torch.Generator().manual_seed(5)
        self.gemm, self.rng = gemm, np.random.default_rng(3)
        self.rows = AttnRows(HEADS, KV_HEADS, DIM, ROT, gated=True)
        self.x_of = torch.randn((VOCAB, self.rows.rows), generator=g).cuda()
        self.logits_of = (torch.randn((VOCAB, VOCAB), generator=g) * 3).cuda()
        self.norm = torch.ones(DIM, device="cuda")
        self.inv_freq = _dev(1e4 ** (-np.arange(ROT // 2) / (ROT // 2)), torch.float32)
        self.kv, self.pool = new_cache(fmt, KV_HEADS, DIM, PAGE, pages), KvPool.new(PAGE, pages, N_SEQ, WIDTH)
        self.text = [[] for _ in range(N_SEQ)]
        self.len = torch.zeros(N_SEQ, dtype=I32, device="cuda")
        self.temp = _dev(np.array([0.8, 0.0, 1.2], np.float32))

    def buffers(self, n, masks=None):
        new = lambda *shape, dtype=I32: torch.full(shape, 77, dtype=dtype, device="cuda")  # noqa: E731
        b = dict(n=n, add=new(N_SEQ), x=new(1, n, self.rows.rows, dtype=torch.float32), start=new(N_SEQ + 1), slots=new(n), pos=new(n),
                 granted=new(N_SEQ), q=new(n, HEADS, DIM, dtype=BF16), gate=new(n, HEADS, DIM, dtype=BF16), out=new(n, HEADS, DIM, dtype=BF16),
                 tokens=new(n), logits=new(n, VOCAB, dtype=torch.float32), u=new(n, 2, dtype=torch.float32), next=new(N_SEQ), count=new(N_SEQ),
                 emit=new(n), src=new(n), dst=new(n), new_len=new(N_SEQ), masks=None if masks is None else _dev(masks.view(np.int64)))
        b["step"] = TreeStep(n, b["start"], self.len, self.pool.table, n if masks is None else len(MASKS), b["masks"])
        return b

    def fill(self, b, news):
        """The step's inputs, from the host: tokens news[seq]."""
        flat = np.concatenate([np.asarray(t, np.int64) for t in news] + [np.zeros(b["n"], np.int64)])[:b["n"]]
        b["add"].copy_(_dev(np.array([len(t) for t in news], np.int32)))
        b["tokens"].copy_(_dev(flat.astype(np.int32)))
        b["x"][0].copy_(self.x_of[_dev(flat)])
        b["logits"].copy_(self.logits_of[_dev(flat)])

    def prompt(self, stream, b):
        kv_plan(stream, self.pool, self.len, b["add"], b["n"], b["start"], b["slots"], b["pos"], b["granted"], mask=b["masks"])
        attn_prep(stream, b["x"], 1, b["n"], self.rows, self.norm, self.norm, self.inv_freq, b["pos"], b["q"], b["gate"], kv=self.kv,
                  slots=b["slots"])
        attend = self.gemm.chunk_attn if b["masks"] is None else self.gemm.tree_attn
        attend(stream, b["q"], HEADS, self.kv, b["step"], b["out"], b["gate"])

    def decode(self, stream, b):
        self.prompt(stream, b)
        self.gemm.verify(stream, b["logits"], VOCAB, b["step"], PAGE, b["tokens"], b["u"], b["next"], b["count"], b["emit"],
                         temp=self.temp, src=b["src"], dst=b["dst"], new_len=b["new_len"])
        kv_move(stream, self.kv, b["src"], b["dst"], b["start"], N_SEQ)
        kv_release(stream, self.pool, b["new_len"])

    def written_in_order(self, news, depths):
        """Every text and the tokens after it in a cache of its own: (cache, slots of each text, queries and gates of all)."""
        kv = KvCache.new(self.kv.fmt, KV_HEADS, DIM, PAGE, N_SEQ * WIDTH)
        at = [np.arange(len(t) + len(m)) + s * WIDTH * PAGE for s, (t, m) in enumerate(zip(self.text, news))]
        pos = [np.r_[np.arange(len(t)), len(t) + np.asarray(d, int)] for t, d in zip(self.text, depths)]
        flat = np.concatenate([np.r_[t, m].astype(np.int64) for t, m in zip(self.text, news)])
        q, gate = torch.empty((2, len(flat), HEADS, DIM), dtype=BF16, device="cuda")
        if len(flat):
            attn_prep(None, self.x_of[_dev(flat)][None], 1, len(flat), self.rows, self.norm, self.norm, self.inv_freq,
                      _dev(np.concatenate(pos).astype(np.int32)), q, gate, kv=kv, slots=_dev(np.concatenate(at).astype(np.int32)))
        return kv, at, q, gate

    def check_attention(self, b, news, depths=None):
        """The step's outputs, those of sequences that were given pages."""
        news = [m if ok else [] for m, ok in zip(news, b["granted"].tolist())]
        depths = depths or [range(len(m)) for m in news]
        first = np.cumsum([0] + [len(t) + len(m) for t, m in zip(self.text, news)])
        s = object.__new__(Chunk if b["masks"] is None else Step)
        s.kv, s.slots, q, gate = self.written_in_order(news, [d[:len(m)] for d, m in zip(depths, news)])
        s.seqs, s.h, s.j, s.d = [(len(t), len(m)) for t, m in zip(self.text, news)], HEADS, KV_HEADS, DIM
        mine = np.concatenate([np.arange(first[k] + len(t), first[k + 1]) for k, t in enumerate(self.text)])
        s.n, s.q, s.gate = len(mine), q[_dev(mine)], gate[_dev(mine)]
        s.start = np.cumsum([0] + [len(m) for m in news])
        s.mask = None if b["masks"] is None else b["masks"].cpu().numpy().view(np.uint64)
        start = b["start"].tolist()
        rows = np.concatenate([np.arange(start[k], start[k] + len(m)) for k, m in enumerate(news)]).astype(np.int64)
        assert torch.equal(b["q"][_dev(rows)], s.q) and torch.equal(b["gate"][_dev(rows)], s.gate)
        out, tol = s.want()
        off = np.abs(_f64(b["out"][_dev(rows)]) - out) - tol
        assert (off <= 0).all(), off.max()

    def check_cache(self):
        kv, at, _, _ = self.written_in_order([[]] * N_SEQ, [[]] * N_SEQ)
        want, got, table = Host(kv), Host(self.kv), self.pool.table.cpu().numpy().astype(np.int64)
        held = self.pool.held.tolist()
        for k, t in enumerate(self.text):
            assert held[k] == -(-len(t) // PAGE)
            p = np.arange(len(t))
            slots = table[k][p // PAGE] * PAGE + p % PAGE
            assert np.array_equal(got.codes[slots], want.codes[at[k]]) and np.array_equal(got.scales[slots], want.scales[at[k]])
        used = np.concatenate([table[k][:h] for k, h in enumerate(held)])
        n = int(self.pool.n_free)
        assert sorted(np.r_[used, self.pool.free.cpu().numpy()[:n]]) == list(range(self.pool.pages))  # each page once

    def walk(self, tokens, u, temp):
        """The path that is kept, and the token after it."""
        path = [0]
        while True:
            row = path[-1]
            y = _choose(_chances(self.logits_of[tokens[row]].cpu().numpy(), temp), u[row, 1])
            child = [k for k, p in enumerate(PARENTS) if p == row and tokens[k] == y]
            if not child:
                return path, y
            path.append(child[0])


@pytest.mark.parametrize("fmt", list(KvFmt))
def test_a_server_run(gemm, fmt):
    s = Server(gemm, fmt, pages=10)
    stream = torch.cuda.Stream()
    random = lambda n: [int(t) for t in s.rng.integers(VOCAB, size=n)]  # noqa: E731

    def chunks(news):
        b = s.buffers(sum(map(len, news)) + 3)  # (three tokens behind the last sequence)
        s.fill(b, news)
        torch.cuda.synchronize()
        b["out"].fill_(77.0)
        with torch.cuda.stream(stream):
            s.prompt(stream, b)
        torch.cuda.synchronize()
        s.check_attention(b, news)
        for k, ok in enumerate(b["granted"].tolist()):
            s.text[k] += news[k] if ok else []
        s.len.copy_(_dev(np.array([len(t) for t in s.text], np.int32)))
        s.check_cache()
        return b["granted"].tolist()

    print(f"prompts {fmt!r}", flush=True)
    assert chunks([random(130), random(1), random(200)]) == [1, 1, 1]  # 3 + 1 + 4 of 10 pages
    assert chunks([random(57), random(300), random(50)]) == [1, 0, 1]  # 0 + 5 pages: the second waits
    assert chunks([[], random(100), []]) == [1, 1, 1]

    # decoding: one graph, replayed over buffers that hold the next step's inputs
    n = N_SEQ * len(MASKS)
    b = s.buffers(n, np.array(MASKS * N_SEQ, np.uint64))
    with torch.cuda.stream(stream):
        graph = Graph.capture(stream, lambda: s.decode(stream, b))
    last = [t[-1] for t in s.text]
    kept, waits = [], 0
    for turn in range(8):
        print(f"trees {turn}", flush=True)
        if turn == 4:  # the third ends, and another request takes its place
            s.text[2] = []
            s.len[2] = 0
            kv_release(None, s.pool, s.len)
            s.check_cache()
            assert chunks([[], [], random(150)]) == [1, 1, 1]
            last[2] = s.text[2][-1]
        u = s.rng.random((n, 2)).astype(np.float32)
        temps = s.temp.cpu().numpy()
        news = []
        for k in range(N_SEQ):
            t, mine = [last[k]] + random(len(MASKS) - 1), u[k * len(MASKS):]
            for i in range(1, len(MASKS)):  # most follow what their parent's row will choose: by the first child, or by the second
                if s.rng.random() < 0.7 and not (i == 1 and turn % 2):
                    t[i] = _choose(_chances(s.logits_of[t[PARENTS[i]]].cpu().numpy(), temps[k]), mine[PARENTS[i], 1])
            news.append(t)
        s.fill(b, news)
        free = int(s.pool.n_free)
        b["u"].copy_(_dev(u))
        torch.cuda.synchronize()
        graph.launch(stream)
        torch.cuda.synchronize()
        need = [-(-(len(t) + len(MASKS)) // PAGE) for t in s.text]
        more = np.cumsum([w - -(-len(t) // PAGE) for w, t in zip(need, s.text)])
        granted = [int(w <= -(-len(t) // PAGE) or m <= free) for w, t, m in zip(need, s.text, more)]
        assert b["granted"].tolist() == granted
        waits += granted.count(0)
        s.check_attention(b, news, [DEPTHS] * N_SEQ)
        for k in range(N_SEQ):
            if not granted[k]:  # it stays as it was
                b["new_len"][k] = s.len[k]
                continue
            path, y = s.walk(news[k], u[k * len(MASKS):], temps[k])
            kept.append(len(path))
            said = [news[k][i] for i in path[1:]] + [y]
            assert b["count"].tolist()[k] == len(path) - 1 and b["next"].tolist()[k] == y
            assert b["emit"][k * len(MASKS):][:len(MASKS)].tolist() == said + [-1] * (len(MASKS) - len(said))
            s.text[k] += [news[k][i] for i in path]
            last[k] = y
        s.len.copy_(b["new_len"])
        assert s.len.tolist() == [len(t) for t in s.text]
        s.check_cache()
    assert set(kept) == {1, 2, 3} and waits
    graph.close()
