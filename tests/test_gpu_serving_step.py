"""A server's step as a whole: plan, rotated append, attention over either cache, the
head's product and the log probabilities of its logits, on device-held state, eagerly,
captured, on two streams."""
import numpy as np
import pytest

import siphon_amd as sa
from siphon_amd import synth

from . import kv4_oracle as k4
from . import kv_oracle as ko
from .test_gpu_logprobs import definition
from .test_gpu_slices import _HipGraph
from .test_gpu_streams import _Streams

pytestmark = pytest.mark.gpu


class Server:
    """One layer for up to n_req requests; the host's copy runs beside it."""

    def __init__(self, dev, seed, bits=4, n_req=5, heads=8, n_kv=2, hd=64, block=16, n_pages=150, max_blocks=30, n_tok=120, max_q=70,
                 vocab=1000, n_top=6, neighbours=False, rot=64, workspace=True):
        self.dev, self.rng, self.bits = dev, np.random.default_rng(seed), bits
        self.n_req, self.heads, self.n_kv, self.hd, self.block = n_req, heads, n_kv, hd, block
        self.n_tok, self.max_q, self.vocab, self.n_top, self.neighbours = n_tok, max_q, vocab, n_top, neighbours
        self.kq = 1 / np.sqrt(hd)
        self.mod = k4 if bits == 4 else ko
        self.cache = self.mod.Cache(self.rng, n_pages, n_kv, hd, block)
        self.table = np.full((n_req, max_blocks), -7, np.int32)
        self.free, self.n_free = self.rng.permutation(n_pages).astype(np.int32), n_pages
        self.length = np.zeros(n_req, np.int32)
        self.rope = k4.table(max_blocks * block, rot)
        z, f = np.zeros, np.float32
        self.d = d = ko.OnDevice(
            dev, table=self.table, free=self.free, len0=self.length, len1=self.length, add=z(n_req, np.int32),
            free0=np.array([n_pages], np.int32), free1=z(1, np.int32), q_start=z(n_req + 1, np.int32), slot=z(n_tok, np.int64),
            pos=z(n_tok, np.int32), status=z(1, np.int32), newk=z((n_tok, n_kv * hd), f), newv=z((n_tok, n_kv * hd), f),
            q=z((n_tok, heads * hd), f), qr=z((n_tok, heads * hd), f), out=z((n_tok, heads * hd), f), rope=self.rope,
            logits=z((n_tok, vocab), f), token=z((n_tok, 1), np.int32), lp=z((n_tok, 1), f), h=z(n_tok, f),
            ti=z((n_tok, n_top), np.int32), tl=z((n_tok, n_top), f))
        self.c = self.mod.put_cache(d, self.cache)
        # (F16 takes any number of rows of any length of whole blocks)
        self.w = dev.upload(sa.F16, vocab, heads * hd, synth.make_weights(sa.F16, vocab, heads * hd, self.rng))
        self.w.prepare_gemm()
        self.attn = sa.AttnPaged(q=d.ptr("qr"), ldq=heads * hd, out=d.ptr("out"), ldo=heads * hd, n_head=heads, kq_scale=self.kq)
        self.args = sa.Logprobs(logits=d.ptr("logits"), ld=vocab, n_rows=n_tok, n_vocab=vocab, token=d.ptr("token"), n_token=1,
                                logprob=d.ptr("lp"), entropy=d.ptr("h"), n_top=n_top, top_id=d.ptr("ti"), top_logprob=d.ptr("tl"))
        if workspace:
            four = bits == 4
            n = (dev.attn_paged4_workspace if four else dev.attn_paged_workspace)(self.c, self.batch(0), self.attn)
            m = dev.logprobs_workspace(self.args)
            self.attn.workspace, self.attn.workspace_bytes = d.put("ws", np.zeros(n, np.uint8)), n
            if m:
                self.args.workspace, self.args.workspace_bytes = d.put("ws2", np.zeros(m, np.uint8)), m

    def batch(self, now):
        p = self.d.ptr
        return sa.KvBatch(q_start=p("q_start"), kv_len=p(f"len{now}"), table=p("table"), n_req=self.n_req,
                          max_blocks=self.table.shape[1], n_tok=self.n_tok, max_q=self.max_q, max_kv=self.table.shape[1] * self.block)

    def enqueue(self, turn, stream=None):
        p, dev, n, w, wide = self.d.ptr, self.dev, 1 - turn, self.n_kv * self.hd, self.heads * self.hd
        dev.kv_plan_dev(sa.KvPlan(len=p(f"len{turn}"), add=p("add"), free_pages=p("free"), n_free=p(f"free{turn}"),
                                  n_req=self.n_req, n_tok=self.n_tok, n_pages=self.cache.n_pages, max_blocks=self.table.shape[1],
                                  block=self.block, table=p("table"), q_start=p("q_start"), kv_len=p(f"len{n}"), slot=p("slot"),
                                  pos=p("pos"), n_free_out=p(f"free{n}"), status=p("status")), stream)
        b = self.batch(n)
        rows = sa.KvRows(k=p("newk"), v=p("newv"), ldk=w, ldv=w, q=p("q"), q_out=p("qr"), ldq=wide, ldq_out=wide, n_head=self.heads,
                         rope=p("rope"), rope_len=len(self.rope), rope_dim=2 * self.rope.shape[1], rope_neighbours=self.neighbours)
        if self.bits == 4:
            dev.kv4_append_dev(self.c, b, rows, stream)
            dev.attn_paged4_dev(self.c, b, self.attn, stream)
        else:
            dev.kv_append_rope_dev(self.c, b, rows, stream)
            dev.attn_paged_dev(self.c, b, self.attn, stream)
        dev.gemm_dev(self.w, p("out"), self.n_tok, p("logits"), stream)
        dev.logprobs_dev(self.args, stream)

    def adds(self, step):
        r, add = self.rng, np.ones(self.n_req, np.int32)
        fresh = self.length == 0
        add[fresh] = r.integers(0, self.max_q + 1, fresh.sum())
        add[~fresh & (r.random(self.n_req) < 0.2)] = -1
        while add[add > 0].sum() > self.n_tok:
            add[np.argmax(add)] //= 2
        return add

    def inputs(self, step):
        r, w = self.rng, self.n_kv * self.hd
        self.add = self.adds(step)
        self.k, self.v = (r.standard_normal((self.n_tok, w)).astype(np.float32) for _ in range(2))
        self.q = r.standard_normal((self.n_tok, self.heads * self.hd)).astype(np.float32) * np.float32(2)
        self.token = r.integers(0, self.vocab, (self.n_tok, 1)).astype(np.int32)
        # rows behind the last token stay as they are: zeros, whose logits are zeros
        for name, a in (("add", self.add), ("newk", self.k), ("newv", self.v), ("q", self.q), ("token", self.token),
                        ("out", np.zeros_like(self.q)), ("qr", np.zeros_like(self.q))):
            self.d.bufs[name][0].fill(a)

    def check(self, turn):
        d, c = self.d, self.cache
        self.table, q_start, kv_len, slot, pos, self.free, self.n_free, status = ko.plan(
            self.length, self.add, self.free, self.n_free, self.table, self.n_tok, self.block)
        assert status == 0 == d.get("status")[0]
        self.length = kv_len
        n = int(q_start[-1])
        turned = lambda x, heads: k4.rotate(x.reshape(self.n_tok, heads, self.hd)[:n], pos[:n], self.rope, self.neighbours)
        q = np.zeros((self.n_tok, self.heads, self.hd), np.float32)
        q[:n] = turned(self.q, self.heads)
        assert np.array_equal(d.get("qr").reshape(q.shape), q)
        c.append(self.table, q_start, kv_len, turned(self.k, self.n_kv), self.v.reshape(self.n_tok, self.n_kv, self.hd)[:n])
        arrays = c.arrays() if self.bits == 4 else {x: getattr(c, x) for x in ("k", "v", "ks", "vs")}
        for name, a in arrays.items():
            assert (d.get(name).view(np.uint8) == np.ascontiguousarray(a).view(np.uint8)).all(), name
        want, err, seen = ko.attention(c, self.table, q_start, kv_len, q, self.kq)
        out = d.get("out").reshape(q.shape)
        assert (out[~seen] == 0).all() and seen.sum() == n
        assert (np.abs(out - want)[seen] <= err[seen] + 1e-30).all()
        # of the logits as they came out (the products have tests of their own)
        x = d.get("logits")
        given, entropy, ids, top, spread = definition(x, self.token, self.n_top)
        bound = (2.0 ** -22 + 3 * spread * 2.0 ** -24) * 65 * (2 + spread)
        assert x[:n].any(1).all() and np.array_equal(d.get("ti"), ids)
        for got, y in ((d.get("lp"), given), (d.get("h")[:, None], entropy[:, None]), (d.get("tl"), top)):
            assert (np.abs(got - y) <= bound[:, None] + 2.0 ** -23 * np.abs(y)).all()

    def close(self):
        self.w.free()
        self.d.__exit__()


@pytest.fixture
def server(dev):
    made = []

    def make(*a, **o):
        made.append(Server(dev, *a, **o))
        return made[-1]

    yield make
    dev.synchronize()
    for s in made:
        s.close()


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("shape", [dict(), dict(heads=4, n_kv=1, hd=128, block=64, n_pages=40, max_blocks=9, neighbours=True, rot=128),
                                   dict(n_req=70, heads=2, n_kv=2, hd=32, block=32, n_pages=500, n_tok=300, rot=20),
                                   dict(heads=4, n_kv=2, hd=96, workspace=False, rot=96, vocab=9000, n_top=20)])
def test_steps(dev, server, bits, shape):
    """Requests start, go on, end and take each other's pages; every byte of the cache is followed."""
    s = server(3, bits, **shape)
    for step in range(8):
        s.inputs(step)
        s.enqueue(step & 1)
        dev.synchronize()
        s.check(step & 1)


@pytest.mark.parametrize("bits", [4, 8])
def test_captured_steps(dev, server, bits):
    """Two steps captured and replayed with other inputs, an eager step of another server between."""
    s, other = server(5, bits), server(6, 12 - bits, workspace=False)
    graphs = [_HipGraph(), _HipGraph()]
    try:
        # (the head's product has its workspace from a call before)
        s.inputs(0)
        s.enqueue(0)
        dev.synchronize()
        s.check(0)
        for turn, g in enumerate(graphs):
            g.begin()
            s.enqueue(turn, g.stream.value)
            g.end()
        for step in range(1, 7):
            s.inputs(step)
            graphs[step & 1].replay()
            s.check(step & 1)
            other.inputs(step)
            other.enqueue(1 - (step & 1))
            dev.synchronize()
            other.check(1 - (step & 1))
    finally:
        for g in graphs:
            g.close()


@pytest.mark.parametrize("own", [True, False])
def test_two_streams(dev, server, own):
    """Two servers step on two streams at once, one with each cache."""
    ss = _Streams()
    try:
        pair = [(server(8 + i, bits, workspace=own), ss.create()) for i, bits in enumerate((4, 8))]
        for step in range(5):
            for s, _ in pair:
                s.inputs(step)
            dev.synchronize()
            for s, stream in pair:
                s.enqueue(step & 1, stream)
            for s, stream in pair:
                ss.sync(stream)
                s.check(step & 1)
    finally:
        dev.synchronize()
        ss.close()
