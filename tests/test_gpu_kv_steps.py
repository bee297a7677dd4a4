"""The calls of the paged 8-bit KV cache together, as a server uses them:
steps on device-held state, captured steps, several streams and graphs."""
import numpy as np
import pytest

import siphon_amd as sa

from . import kv_oracle as ko
from .test_gpu_slices import _HipGraph
from .test_gpu_streams import _Streams

pytestmark = pytest.mark.gpu


class Server:
    """One layer of a model for up to n_req requests: everything a step needs
    stays on the device, the numbers in two copies that take turns. The host's
    copy (kv_oracle) runs beside it."""

    def __init__(self, dev, seed, n_req=6, heads=8, n_kv=2, hd=64, block=16, n_pages=150, max_blocks=40, n_tok=160, max_q=90,
                 workspace=True):
        self.dev, self.rng = dev, np.random.default_rng(seed)
        self.n_req, self.heads, self.n_kv, self.hd, self.block = n_req, heads, n_kv, hd, block
        self.n_tok, self.max_q, self.kq = n_tok, max_q, 1 / np.sqrt(hd)
        self.cache = ko.Cache(self.rng, n_pages, n_kv, hd, block)
        self.table = np.full((n_req, max_blocks), -7, np.int32)
        self.free, self.n_free = self.rng.permutation(n_pages).astype(np.int32), n_pages
        self.length = np.zeros(n_req, np.int32)
        z = np.zeros
        self.d = d = ko.OnDevice(
            dev, table=self.table, free=self.free, len0=self.length, len1=self.length, add=z(n_req, np.int32),
            free0=np.array([n_pages], np.int32), free1=z(1, np.int32), q_start=z(n_req + 1, np.int32), slot=z(n_tok, np.int64),
            pos=z(n_tok, np.int32), status=z(1, np.int32), newk=z((n_tok, n_kv * hd), np.float32),
            newv=z((n_tok, n_kv * hd), np.float32), q=z((n_tok, heads * hd), np.float32), out=z((n_tok, heads * hd), np.float32),
            backk=z((n_tok, n_kv * hd), np.float32), backv=z((n_tok, n_kv * hd), np.float32))
        self.c = ko.put_cache(d, self.cache)
        self.attn = sa.AttnPaged(q=d.ptr("q"), ldq=heads * hd, out=d.ptr("out"), ldo=heads * hd, n_head=heads, kq_scale=self.kq)
        if workspace:
            n = dev.attn_paged_workspace(self.c, self.batch(0), self.attn)
            assert n > 0
            d.put("ws", np.zeros(n, np.uint8))
            self.attn.workspace, self.attn.workspace_bytes = d.ptr("ws"), n

    def batch(self, now):
        p = self.d.ptr
        return sa.KvBatch(q_start=p("q_start"), kv_len=p(f"len{now}"), table=p("table"), n_req=self.n_req,
                          max_blocks=self.table.shape[1], n_tok=self.n_tok, max_q=self.max_q, max_kv=self.table.shape[1] * self.block)

    def enqueue(self, turn, stream=None):
        """A step's calls: numbers of copy `turn` in, of the other out."""
        p, dev, n, w = self.d.ptr, self.dev, 1 - turn, self.n_kv * self.hd
        dev.kv_plan_dev(sa.KvPlan(len=p(f"len{turn}"), add=p("add"), free_pages=p("free"), n_free=p(f"free{turn}"),
                                  n_req=self.n_req, n_tok=self.n_tok, n_pages=self.cache.n_pages, max_blocks=self.table.shape[1],
                                  block=self.block, table=p("table"), q_start=p("q_start"), kv_len=p(f"len{n}"), slot=p("slot"),
                                  pos=p("pos"), n_free_out=p(f"free{n}"), status=p("status")), stream)
        b = self.batch(n)
        dev.kv_append_dev(self.c, b, p("newk"), w, p("newv"), w, stream)
        dev.attn_paged_dev(self.c, b, self.attn, stream)
        dev.kv_read_dev(self.c, p("slot"), self.n_tok, p("backk"), w, p("backv"), w, stream)

    def inputs(self, add):
        r, w = self.rng, self.n_kv * self.hd
        self.add = np.asarray(add, np.int32)
        self.k, self.v = (r.standard_normal((self.n_tok, w)).astype(np.float32) * np.float32(np.exp(r.normal())) for _ in range(2))
        self.q = r.standard_normal((self.n_tok, self.heads * self.hd)).astype(np.float32) * np.float32(2)
        for name, a in (("add", self.add), ("newk", self.k), ("newv", self.v), ("q", self.q),
                        *((x, np.full_like(self.q, 55)) for x in ("out",)),
                        *((x, np.full_like(self.k, 55)) for x in ("backk", "backv"))):
            self.d.bufs[name][0].fill(a)

    def check(self, turn):
        """The step on the host, and everything it left on the device."""
        d, c = self.d, self.cache
        self.table, q_start, kv_len, slot, pos, self.free, self.n_free, status = ko.plan(
            self.length, self.add, self.free, self.n_free, self.table, self.n_tok, self.block)
        assert status == 0 == d.get("status")[0]
        self.length = kv_len
        n = 1 - turn
        for name, want in (("table", self.table), ("q_start", q_start), (f"len{n}", kv_len), ("slot", slot), ("pos", pos),
                           ("free", self.free), (f"free{n}", [self.n_free])):
            assert np.array_equal(d.get(name), want), name
        rows = (self.n_tok, self.n_kv, self.hd)
        c.append(self.table, q_start, kv_len, self.k.reshape(rows), self.v.reshape(rows))
        for name in ("k", "v", "ks", "vs"):
            assert np.array_equal(d.get(name).view(np.uint8), getattr(c, name).view(np.uint8)), name
        q = self.q.reshape(self.n_tok, self.heads, self.hd)
        want, err, seen = ko.attention(c, self.table, q_start, kv_len, q, self.kq)
        got = d.get("out").reshape(q.shape)
        assert (got[~seen] == 55).all() and seen.sum() == q_start[-1]
        assert (np.abs(got - want)[seen] <= err[seen] + 1e-30).all()
        for name, codes, scales in (("backk", c.k, c.ks), ("backv", c.v.swapaxes(2, 3), c.vs)):
            back, at = d.get(name).reshape(rows), slot[seen]
            page = at // self.block
            x = codes[page, :, at % self.block].astype(np.float32) * scales[page][:, :, None]
            assert np.array_equal(back[seen].view(np.uint32), x.view(np.uint32)) and (back[~seen] == 55).all()

    def adds(self, step):
        """Prompts in chunks, single tokens, requests that wait, end, or start
        again on pages of others."""
        r, add = self.rng, np.ones(self.n_req, np.int32)
        fresh = self.length == 0
        add[fresh] = r.integers(0, self.max_q + 1, fresh.sum())
        chunk = ~fresh & (r.random(self.n_req) < 0.2)
        add[chunk] = r.integers(0, 40, chunk.sum())
        add[~fresh & (r.random(self.n_req) < 0.2)] = -1
        while add[add > 0].sum() > self.n_tok:
            add[np.argmax(add)] //= 2
        if step % 7 == 6:
            add[:] = -1
        return add

    def close(self):
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


@pytest.mark.parametrize("shape", [dict(), dict(heads=6, n_kv=1, hd=128, block=64, n_pages=40, max_blocks=12),
                                   dict(n_req=70, heads=2, n_kv=2, hd=48, block=32, n_pages=500, n_tok=700),
                                   dict(heads=4, n_kv=2, hd=256, block=16, workspace=False)])
def test_steps(dev, server, shape):
    """Twenty steps in which requests start, go on, end and take each other's
    pages; every byte of the cache is followed."""
    s = server(3, **shape)
    for step in range(20):
        s.inputs(s.adds(step))
        s.enqueue(step & 1)
        dev.synchronize()
        s.check(step & 1)
    assert s.length.max() > 0


def test_captured_steps(dev, server):
    """Two steps captured into a graph (from one copy of the numbers to the
    other and back), replayed with other inputs each time and an eager step's
    calls of another server between the replays."""
    s, other = server(5), server(6, workspace=False)
    hg = _HipGraph()
    try:
        hg.begin()
        s.enqueue(0, hg.stream.value)
        hg.end()
        back = _HipGraph()
        try:
            back.begin()
            s.enqueue(1, back.stream.value)
            back.end()
            for step in range(10):
                s.inputs(s.adds(step))
                (back if step & 1 else hg).replay()
                s.check(step & 1)
                other.inputs(other.adds(step))
                other.enqueue(step & 1)
                dev.synchronize()
                other.check(step & 1)
        finally:
            back.close()
    finally:
        hg.close()


def test_capture_without_a_workspace_is_refused_when_it_must_grow(dev, server):
    """The context's workspace cannot grow in a capture; a call that needs
    none, or has its own, is captured."""
    ctx2 = sa.Device(0)
    try:
        s = Server(ctx2, 7, workspace=False)
        hg = _HipGraph()
        try:
            hg.begin()
            with pytest.raises(sa.SihipError, match="capture"):
                ctx2.attn_paged_dev(s.c, s.batch(1), s.attn, hg.stream.value)
            hg.end()
        finally:
            hg.close()
        s.inputs(s.adds(0))
        s.enqueue(0)
        ctx2.synchronize()
        s.check(0)
        s.close()
    finally:
        ctx2.close()


@pytest.mark.parametrize("own", [True, False])
def test_two_streams(dev, server, own):
    """Two servers step on two streams at once, with workspaces of their own
    or with the context's in turns."""
    ss = _Streams()
    try:
        pair = [(server(8 + i, workspace=own), ss.create()) for i in range(2)]
        for step in range(6):
            for s, _ in pair:
                s.inputs(s.adds(step))
            dev.synchronize()
            for s, stream in pair:
                s.enqueue(step & 1, stream)
            for s, stream in pair:
                ss.sync(stream)
                s.check(step & 1)
    finally:
        dev.synchronize()
        ss.close()


def test_two_graphs_at_once(dev, server):
    """Two captured steps with workspaces of their own, replayed at once."""
    graphs = []
    try:
        pair = [server(20 + i) for i in range(2)]
        for s in pair:
            g = _HipGraph()
            graphs.append(g)
            g.begin()
            s.enqueue(0, g.stream.value)
            g.end()
        for step in range(4):
            for s in pair:
                # numbers of copy 1 become copy 0's: the graph steps from 0 to 1
                for name, a in (("len0", s.length), ("free0", np.array([s.n_free], np.int32))):
                    s.d.bufs[name][0].fill(a)
                s.inputs(s.adds(step))
            dev.synchronize()
            for g in graphs:
                g._ok(g.hip.hipGraphLaunch(g.exec, g.stream))
            for g in graphs:
                g._ok(g.hip.hipStreamSynchronize(g.stream))
            for s in pair:
                s.check(0)
    finally:
        for g in graphs:
            g.close()


def test_one_workspace_for_calls_of_any_size(dev):
    """A workspace that was zeroed once serves calls of any shapes one after
    the other: its counters are zero after each."""
    rng = np.random.default_rng(30)
    shapes = [([3000, 100], [1, 1], 8, 2, 128), ([500, 0], [200, 300], 4, 2, 128), ([9000], [1], 4, 4, 64), ([40] * 20, [2] * 20, 3, 1, 32),
              ([700, 2500, 0], [100, 1, 9], 2, 2, 256), ([3000, 100], [1, 1], 8, 2, 128)]
    ws = dev.to_device(np.zeros(64 << 20, np.uint8))
    try:
        for lengths, adds, heads, n_kv, hd in shapes * 2:
            cache, table, q_start, kv_len = ko.requests(rng, lengths, adds, 32, n_kv, hd)
            n = int(q_start[-1])
            q = rng.standard_normal((n, heads, hd)).astype(np.float32)
            with ko.OnDevice(dev, q=q, out=np.zeros_like(q)) as d:
                c, b = ko.put_cache(d, cache), ko.put_batch(d, table, q_start, kv_len, n)
                a = sa.AttnPaged(q=d.ptr("q"), ldq=heads * hd, out=d.ptr("out"), ldo=heads * hd, n_head=heads, kq_scale=0.1,
                                 workspace=ws.ptr, workspace_bytes=ws.nbytes)
                assert dev.attn_paged_workspace(c, b, a) <= ws.nbytes
                dev.attn_paged_dev(c, b, a)
                dev.synchronize()
                want, err, _ = ko.attention(cache, table, q_start, kv_len, q, 0.1)
                assert (np.abs(d.get("out") - want) <= err + 1e-30).all()
            assert not ws.to_host(np.uint32, 1 << 16).any()
    finally:
        ws.free()


def test_another_device_context(dev):
    """Two contexts of the device hold caches of their own and step at once."""
    ctx2 = sa.Device(0)
    try:
        a, b = Server(dev, 40, workspace=False), Server(ctx2, 41, workspace=False)
        for step in range(4):
            for s in (a, b):
                s.inputs(s.adds(step))
            for s in (a, b):
                s.enqueue(step & 1)
            dev.synchronize()
            ctx2.synchronize()
            for s in (a, b):
                s.check(step & 1)
        a.close()
        b.close()
    finally:
        ctx2.close()


def bits(a):
    return np.ascontiguousarray(a).view(np.uint32)


@pytest.mark.parametrize("start", [0, 1, 7, 15, 16, 40])
@pytest.mark.parametrize("block,n_kv,hd,wide", [(16, 2, 64, True), (32, 1, 16, True), (64, 2, 80, False), (16, 1, 48, False),
                                                (32, 16, 64, True)])
def test_read_runs(dev, block, n_kv, hd, wide, start):
    """Slots that go on from one another over pages in any order, from any
    place in a page, the last group ragged; aligned rows and odd ones."""
    rng = np.random.default_rng(block + hd + start)
    n = 2100 if n_kv == 16 else 205
    cache, table, _, _ = ko.requests(rng, [start + n], [0], block, n_kv, hd)
    k, v = cache.rows(table[0], start + n)
    at = np.arange(start, start + n)
    slots = table[0, at // block].astype(np.int64) * block + at % block
    ld, shift = (n_kv * hd + 4, 4) if wide else (n_kv * hd + 1, 1)
    marker = np.full(n * ld + shift, 55.0, np.float32)
    with ko.OnDevice(dev, slots=slots, ko=marker, vo=marker) as d:
        dev.kv_read_dev(ko.put_cache(d, cache), d.ptr("slots"), n, d.ptr("ko") + 4 * shift, ld, d.ptr("vo") + 4 * shift, ld)
        dev.synchronize()
        for name, x in (("ko", k), ("vo", v)):
            want = np.full((n, ld), 55.0, np.float32)
            want[:, :n_kv * hd] = x.swapaxes(0, 1)[start:].reshape(n, -1).astype(np.float32)
            got = d.get(name)
            assert (got[:shift] == 55).all()
            assert np.array_equal(bits(got[shift:].reshape(n, ld)), bits(want))
