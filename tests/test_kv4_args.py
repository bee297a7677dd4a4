"""What the calls of the 4-bit KV cache, of rotated appends and of log probabilities
refuse, and what they launch, on the CPU (host/fake_hip.cpp): nothing here runs a kernel."""
import pytest

from . import fake_hip
from .test_kv_args import SETUP as SETUP8

SETUP = SETUP8 + """
def cache4(**o):
    return sa.Kv4Cache(**{**dict(k=X, v=X, k_sub=X, v_sub=X, k_scale=X, v_scale=X, n_pages=100, n_head_kv=8, head_dim=128, block=32), **o})
def rows(**o):
    return sa.KvRows(**{**dict(k=X, v=X, ldk=1024, ldv=1024, q=X, q_out=X, ldq=4096, ldq_out=4096, n_head=32, rope=X, rope_len=640,
                               rope_dim=128), **o})
def lp(**o):
    return sa.Logprobs(**{**dict(logits=X, ld=5000, n_rows=3, n_vocab=5000, token=X, n_token=1, logprob=X, entropy=X, n_top=5, top_id=X,
                                 top_logprob=X), **o})
fake.fake_reset(0)
"""


def errors(lines):
    got = fake_hip.run(SETUP + "result = [" + ", ".join(f"said({x})" for x in lines) + "]\n"
                       "result.append(launched())")
    assert got.pop() == [], "a refused call launched something"
    return dict(zip(lines, got))


def refused(lines):
    for line, text in errors(list(lines)).items():
        assert "error -5" in text and lines[line] in text, (line, text)


CALLS4 = ["dev.kv4_append_dev, {}, batch(), rows()", "dev.kv4_read_dev, {}, X, 4, X, 4096, X, 4096", "dev.attn_paged4_dev, {}, batch(), attn()",
          "dev.attn_paged4_workspace, {}, batch(), attn()"]


def test_bad_caches_are_refused_by_every_call():
    bad = {**{f"{n}=0": "NULL" for n in ("k", "v", "k_sub", "v_sub", "k_scale", "v_scale")},
           **{f"{n}=X + 8": "aligned" for n in ("k", "v", "k_sub", "v_sub", "k_scale", "v_scale")},
           "block=8": "block", "block=48": "block", "block=512": "block", "block=0": "block", "head_dim=0": "head_dim",
           "head_dim=16": "head_dim", "head_dim=80": "head_dim", "head_dim=288": "head_dim", "n_head_kv=0": "n_head_kv",
           "n_head_kv=4097": "n_head_kv", "n_pages=0": "n_pages", "n_pages=1 << 31": "n_pages"}
    refused({c.format(f"cache4({b})"): w for b, w in bad.items() for c in CALLS4})


def test_bad_batches_are_refused():
    bad = {"q_start=0": "NULL", "kv_len=0": "NULL", "table=0": "NULL", "n_req=0": "n_req", "n_req=4097": "n_req",
           "max_blocks=0": "max_blocks", "max_blocks=1 << 27": "max_blocks", "n_tok=-1": "n_tok", "n_tok=1 << 31": "n_tok",
           "max_q=-1": "max_q", "max_kv=-1": "max_kv"}
    calls = ["dev.kv4_append_dev, cache4(), batch({}), rows()", "dev.kv_append_rope_dev, cache(), batch({}), rows()",
             "dev.attn_paged4_dev, cache4(), batch({}), attn()"]
    refused({c.format(b): w for b, w in bad.items() for c in calls})


def test_bad_rows_are_refused():
    bad = {"k=0": "f32", "v=X + 2": "f32", "ldk=1023": "ldk", "ldv=0": "ldv", "rope_dim=0": "rope_dim", "rope_dim=-2": "rope_dim",
           "rope_dim=127": "rope_dim", "rope_dim=130": "rope_dim", "rope_len=639": "rope_len", "rope_len=0": "rope_len",
           "rope=X + 2": "f32", "q_out=0": "f32", "q_out=X + 2": "f32", "q=X + 1": "f32", "n_head=0": "n_head", "n_head=20": "n_head",
           "n_head=4104": "n_head", "n_head=1 << 62": "n_head", "ldq=4095": "ldq", "ldq_out=100": "ldq", "ldq_out=8192": "in place"}
    calls = ["dev.kv4_append_dev, cache4(), batch(), rows({})", "dev.kv_append_rope_dev, cache(), batch(), rows({})"]
    refused({**{c.format(b): w for b, w in bad.items() for c in calls},
             "dev.kv_append_rope_dev, cache(), batch(), rows(rope=0, q=0)": "rope",
             "dev.kv4_append_dev, cache4(), batch(), rows(rope=0)": "without a rotation",
             "dev.kv4_read_dev, cache4(), 0, 4, X, 4096, X, 4096": "slots", "dev.kv4_read_dev, cache4(), X + 4, 4, X, 4096, X, 4096": "slots",
             "dev.kv4_read_dev, cache4(), X, -1, X, 4096, X, 4096": "rows", "dev.kv4_read_dev, cache4(), X, 4, X, 1023, X, 4096": "rows",
             "dev.kv4_read_dev, cache4(), X, 4, X, 4096, 0, 4096": "f32",
             **{f"dev.attn_paged4_dev, cache4(), batch(), attn({b})": "attn_paged4" for b in (
                 "q=0", "out=0", "out=X + 2", "n_head=0", "n_head=20", "n_head=4104", "ldq=4095", "ldo=100",
                 "kq_scale=float('nan')", "kq_scale=float('inf')", "softcap=-1.0", "softcap=float('nan')", "window=-1")}})


def test_a_table_of_the_batch_is_enough():
    """Positions end at max_kv, or where the table's rows do."""
    got = fake_hip.run(SETUP + """
dev.kv4_append_dev(cache4(), batch(max_kv=100), rows(rope_len=100))
dev.kv4_append_dev(cache4(), batch(max_kv=10 ** 6), rows(rope_len=640))
dev.kv4_append_dev(cache4(), batch(), rows(rope=0, rope_len=0, rope_dim=0, q=0))
dev.kv_append_rope_dev(cache(), batch(), rows(q=0, q_out=0))
result = launched()
""")
    assert [k for k, *_ in got] == ["kv4_append_kernel"] * 3 + ["kv_append_kernel<1,256,sihip::KeyRope>"]


def test_bad_logprobs_are_refused():
    bad = {"logits=0": "NULL logits", "logits=X + 2": "aligned", "ld=4999": "ld", "n_rows=-1": "rows", "n_rows=1 << 24": "rows",
           "n_vocab=0": "logits", "n_vocab=1 << 31, ld=1 << 32": "logits", "n_token=-1": "n_token", "n_top=-1": "n_top", "n_top=65": "n_top",
           "n_vocab=4, ld=4": "n_top", "token=0": "together", "logprob=0": "together", "top_id=0": "top_id", "top_logprob=0": "top_id",
           "entropy=X + 1": "aligned", "top_id=X + 3": "aligned"}
    refused({f"dev.logprobs_dev, lp({b})": w for b, w in bad.items()})


def test_nothing_to_do_launches_nothing():
    got = fake_hip.run(SETUP + """
dev.kv4_append_dev(cache4(), batch(max_q=0), rows(k=0, v=0))
dev.kv4_append_dev(cache4(), batch(n_tok=0), rows(k=0, v=0))
dev.kv_append_rope_dev(cache(), batch(n_tok=0), rows(k=0, v=0))
dev.kv4_read_dev(cache4(), 0, 0, 0, 4096, 0, 4096)
dev.attn_paged4_dev(cache4(), batch(n_tok=0), attn(q=0, out=0))
dev.logprobs_dev(lp(n_rows=0, logits=0))
result = launched()
""")
    assert got == []


@pytest.mark.parametrize("call", ["attn", "logprobs"])
@pytest.mark.parametrize("what", ["small", "exact", "aligned", "capture"])
def test_workspaces(what, call):
    """A caller's workspace must be as large as asked for; the context's must
    exist before a capture."""
    got = fake_hip.run(SETUP + f"""
what = {what!r}
if {call!r} == "attn":
    c, b = cache4(), batch(max_kv=2000, max_blocks=80, n_tok=1, n_req=1)
    n = dev.attn_paged4_workspace(c, b, attn())
    go = lambda stream=None, **o: said(dev.attn_paged4_dev, c, b, attn(**o), stream)
else:
    n = dev.logprobs_workspace(lp(n_vocab=50000, ld=50000))
    go = lambda stream=None, **o: said(dev.logprobs_dev, lp(n_vocab=50000, ld=50000, **o), stream)
if what == "capture":
    fake.fake_capture(1)
    first = go(5)
    fake.fake_capture(0)
    go(5)
    fake.fake_capture(1)
    result = [n, first, go(5)]
else:
    size, at = dict(small=(n - 1, X), exact=(n, X), aligned=(n + 512, X + 8))[what]
    result = [n, go(workspace=at, workspace_bytes=size)]
""")
    assert got[0] > 0
    if what == "exact":
        assert got[1] == ""
    elif what == "capture":
        assert "capture" in got[1] and got[2] == ""
    else:
        assert "workspace" in got[1]


def test_the_splits_of_rows():
    """Few rows are split until the device is full, many are not."""
    got = fake_hip.run(SETUP + """
for rows_, n in ((1, 1), (1, 4000), (1, 151936), (64, 32003), (500, 151936), (2048, 151936), (1, 2 ** 31 - 1)):
    dev.logprobs_dev(lp(n_rows=rows_, n_vocab=n, ld=n, n_top=min(n, 5)))
dev.logprobs_dev(lp(n_top=0))
result = launched()
""")
    assert [g[:2] for g in got] == [["logprobs_kernel<true>", g] for g in (1, 1, 38, 512, 1000, 2048, 64)] + [["logprobs_kernel<false>", 6]]


def test_a_failed_launch_is_reported():
    for call in ("kv4_append_dev(cache4(), batch(), rows())", "kv_append_rope_dev(cache(), batch(), rows())",
                 "kv4_read_dev(cache4(), X, 4, X, 4096, X, 4096)", "attn_paged4_dev(cache4(), batch(), attn())", "logprobs_dev(lp())"):
        got = fake_hip.run(SETUP + f"""
fake.fake_reset(1)
try:
    dev.{call}
    result = ""
except sa.SihipError as e:
    result = str(e)
""")
        assert "error -8" in got, call


@pytest.mark.parametrize("step,want", [
    # (tokens, requests, longest, heads, KV heads, head_dim, most tokens of a request)
    ((1, 1, 600, 32, 8, 128, 1), [["attnp4_groups_kernel<32,1,8,4,4,4>", 264, 1]]),
    ((64, 64, 8192, 32, 8, 128, 1), [["attnp4_groups_kernel<32,1,8,4,4,4>", 1280, 1]]),
    ((256, 256, 8192, 32, 8, 128, 1), [["attnp4_groups_kernel<32,1,8,4,1,4>", 4096, 1]]),
    ((2, 1, 600, 8, 8, 128, 2), [["attnp4_groups_kernel<32,1,8,4,4,4>", 264, 1]]),
    ((1, 1, 600, 14, 2, 64, 1), [["attnp4_groups_kernel<16,1,4,4,4,2>", 258, 1]]),
    ((1, 1, 600, 2, 1, 192, 1), [["attnp4_groups_kernel<32,2,12,2,4,8>", 257, 1]]),
    ((1, 1, 600, 2, 1, 256, 1), [["attnp4_groups_kernel<32,2,16,2,4,8>", 257, 1]]),
    # more rows than columns for their groups
    ((1, 1, 600, 16, 1, 64, 1), [["attnp4_rows_kernel<16,1,4,4,4>", 257, 1]]),
    ((1, 1, 600, 5, 1, 128, 1), [["attnp4_rows_kernel<32,1,8,4,4>", 257, 1]]),
    ((1, 1, 600, 3, 1, 256, 1), [["attnp4_rows_kernel<32,2,16,2,4>", 257, 1]]),
    ((509, 1, 509, 14, 2, 64, 509), [["attnp4_rows_kernel<16,1,4,4,4>", 446, 1]]),
    ((4096, 1, 4096, 32, 8, 256, 4096), [["attnp4_rows_kernel<32,2,16,2,1>", 9216, 1]]),
    # large row blocks, the shorter requests beside them, splits of their keys
    ((4096, 1, 4096, 32, 8, 128, 4096), [["attnp4_tiles_kernel<8,8>", 512, 1]]),
    ((4096, 1, 4096, 32, 8, 96, 4096), [["attnp4_tiles_kernel<6,8>", 512, 1]]),
    ((4096, 1, 4096, 32, 8, 64, 4096), [["attnp4_tiles_kernel<4,4>", 1024, 1]]),
    ((1100, 65, 16000, 32, 8, 128, 1024), [["attnp4_tiles_kernel<8,8>", 656, 1], ["attnp4_rows_kernel<32,1,8,4,1>", 3104, 1]]),
    ((256, 1, 64000, 32, 8, 128, 256), [["attnp4_tiles_kernel<8,8>", 32, 8], ["attnp_join_kernel<256>", 32, 32]]),
])
def test_kernels_of_attention(step, want):
    n_tok, n_req, longest, heads, n_kv, hd, max_q = step
    assert fake_hip.run(SETUP + f"""
dev.attn_paged4_dev(cache4(n_head_kv={n_kv}, head_dim={hd}, block=64, n_pages=10000),
                    batch(n_tok={n_tok}, n_req={n_req}, max_q={max_q}, max_kv={longest}, max_blocks=4096),
                    attn(n_head={heads}, ldq={heads * hd}, ldo={heads * hd}))
result = launched()
""") == want


@pytest.mark.parametrize("block,hd,want", [(16, 64, "1,128"), (16, 256, "1,256"), (64, 128, "1,512"), (64, 256, "1,1024"),
                                           (256, 128, "2,1024"), (256, 256, "4,1024")])
def test_kernels_of_rotated_appends(block, hd, want):
    """Of the 8-bit cache by the page's units of 16 codes, a third layer of workgroups for queries."""
    got = fake_hip.run(SETUP + f"""
c = dict(n_head_kv=2, head_dim={hd}, block={block})
r = dict(ldk={2 * hd}, ldv={2 * hd}, n_head=4, ldq={4 * hd}, ldq_out={4 * hd}, rope_dim={hd}, rope_len=20 * {block})
dev.kv_append_rope_dev(cache(**c), batch(max_kv=20 * {block}), rows(**r))
dev.kv4_append_dev(cache4(**c), batch(max_kv=20 * {block}), rows(**r))
result = launched()
""")
    assert got == [[f"kv_append_kernel<{want},sihip::KeyRope>", 2, 4], ["kv4_append_kernel", 2, 4]]
