"""What the calls of the paged KV cache refuse, and what they launch, on the
CPU (host/fake_hip.cpp): nothing here runs a kernel."""
import pytest

from . import fake_hip

SETUP = """
def cache(**o):
    return sa.KvCache(**{**dict(k=X, v=X, k_scale=X, v_scale=X, n_pages=100, n_head_kv=8, head_dim=128, block=32), **o})
def batch(**o):
    return sa.KvBatch(**{**dict(q_start=X, kv_len=X, table=X, n_req=4, max_blocks=20, n_tok=4, max_q=1, max_kv=640), **o})
def plan(**o):
    return sa.KvPlan(**{**dict(len=X, add=X, free_pages=X, n_free=X, n_req=4, n_tok=4, n_pages=100, max_blocks=20,
                               block=32, table=X, q_start=X, kv_len=X + 64, slot=X, pos=X, n_free_out=X + 64, status=X), **o})
def attn(**o):
    return sa.AttnPaged(**{**dict(q=X, ldq=4096, out=X, ldo=4096, n_head=32, kq_scale=0.1), **o})
def said(f, *a):
    try:
        f(*a)
        return ""
    except sa.SihipError as e:
        return str(e)
    except Exception as e:
        return "not an error of the library: %r" % e
fake.fake_reset(0)
"""


def errors(lines):
    got = fake_hip.run(SETUP + "result = [" + ", ".join(f"said({x})" for x in lines) + "]\n"
                       "result.append(launched())")
    assert got.pop() == [], "a refused call launched something"
    return dict(zip(lines, got))


def test_bad_caches_are_refused_by_every_call():
    bad = {"k=0": "NULL", "v=0": "NULL", "k_scale=0": "NULL", "v_scale=0": "NULL", "block=8": "block",
           "block=48": "block", "block=512": "block", "block=0": "block", "head_dim=0": "head_dim",
           "head_dim=24": "head_dim", "head_dim=272": "head_dim", "n_head_kv=0": "n_head_kv",
           "n_head_kv=4097": "n_head_kv", "n_pages=0": "n_pages", "n_pages=1 << 31": "n_pages", "k=X + 8": "aligned",
           "v=X + 1": "aligned", "k_scale=X + 2": "aligned"}
    calls = ["dev.kv_append_dev, cache({}), batch(), X, 4096, X, 4096", "dev.kv_read_dev, cache({}), X, 4, X, 4096, X, 4096",
             "dev.attn_paged_dev, cache({}), batch(), attn()"]
    lines = {c.format(b): w for b, w in bad.items() for c in calls}
    for line, text in errors(list(lines)).items():
        assert "error -5" in text and lines[line] in text, (line, text)


def test_bad_batches_are_refused():
    bad = {"q_start=0": "NULL", "kv_len=0": "NULL", "table=0": "NULL", "n_req=0": "n_req", "n_req=4097": "n_req",
           "max_blocks=0": "max_blocks", "max_blocks=1 << 27": "max_blocks", "n_tok=-1": "n_tok", "n_tok=1 << 31": "n_tok",
           "max_q=-1": "max_q", "max_kv=-1": "max_kv"}
    calls = ["dev.kv_append_dev, cache(), batch({}), X, 4096, X, 4096", "dev.attn_paged_dev, cache(), batch({}), attn()"]
    lines = {c.format(b): w for b, w in bad.items() for c in calls}
    for line, text in errors(list(lines)).items():
        assert "error -5" in text and lines[line] in text, (line, text)


def test_bad_plans_are_refused():
    bad = {**{f"{n}=0": "NULL" for n in ("len", "add", "free_pages", "n_free", "table", "q_start", "kv_len", "slot", "pos",
                                         "n_free_out", "status")},
           "n_req=0": "n_req", "n_req=4097": "n_req", "block=33": "block", "n_tok=-1": "n_tok", "n_tok=1 << 31": "n_tok",
           "n_pages=0": "n_pages", "max_blocks=0": "max_blocks", "max_blocks=1 << 26": "max_blocks",
           "kv_len=X": "inputs", "n_free_out=X": "inputs"}
    lines = {f"dev.kv_plan_dev, plan({b})": w for b, w in bad.items()}
    for line, text in errors(list(lines)).items():
        assert "error -5" in text and lines[line] in text, (line, text)


def test_bad_rows_and_scores_are_refused():
    lines = ["dev.kv_append_dev, cache(), batch(), 0, 4096, X, 4096", "dev.kv_append_dev, cache(), batch(), X, 4096, X + 2, 4096",
             "dev.kv_append_dev, cache(), batch(), X, 1023, X, 4096", "dev.kv_append_dev, cache(), batch(), X, 4096, X, 1023",
             "dev.kv_read_dev, cache(), 0, 4, X, 4096, X, 4096", "dev.kv_read_dev, cache(), X, -1, X, 4096, X, 4096",
             "dev.kv_read_dev, cache(), X + 4, 4, X, 4096, X, 4096", "dev.kv_read_dev, cache(), X, 4, X, 1000, X, 4096",
             "dev.kv_read_dev, cache(), X, 4, X, 4096, 0, 4096",
             *(f"dev.attn_paged_dev, cache(), batch(), attn({b})" for b in (
                 "q=0", "out=0", "out=X + 2", "n_head=0", "n_head=20", "n_head=4104", "ldq=4095", "ldo=100",
                 "kq_scale=float('nan')", "kq_scale=float('inf')", "softcap=-1.0", "softcap=float('nan')", "window=-1"))]
    for line, text in errors(lines).items():
        assert "error -5" in text, (line, text)


def test_nothing_to_do_launches_nothing():
    got = fake_hip.run(SETUP + """
dev.kv_append_dev(cache(), batch(max_q=0), 0, 4096, 0, 4096)
dev.kv_append_dev(cache(), batch(n_tok=0), 0, 4096, 0, 4096)
dev.kv_read_dev(cache(), 0, 0, 0, 4096, 0, 4096)
dev.attn_paged_dev(cache(), batch(n_tok=0), attn(q=0, out=0))
result = launched()
""")
    assert got == []
    # a step in which every request ends or waits still has a plan
    got = fake_hip.run(SETUP + "dev.kv_plan_dev(plan(n_tok=0, slot=0, pos=0)); result = launched()")
    assert [k for k, *_ in got] == ["kv_plan_kernel<256>"]


@pytest.mark.parametrize("what", ["small", "exact", "aligned", "capture"])
def test_workspaces(what):
    """A caller's workspace must be as large as asked for; the context's must
    exist before a capture."""
    got = fake_hip.run(SETUP + f"""
what = {what!r}
c, b, a = cache(), batch(max_kv=2000, max_blocks=80, n_tok=1, n_req=1), attn()
n = dev.attn_paged_workspace(c, b, a)
if what == "capture":
    fake.fake_capture(1)
    first = said(dev.attn_paged_dev, c, b, a, 5)
    fake.fake_capture(0)
    dev.attn_paged_dev(c, b, a, 5)
    fake.fake_capture(1)
    result = [n, first, said(dev.attn_paged_dev, c, b, a, 5)]
else:
    size, at = dict(small=(n - 1, X), exact=(n, X), aligned=(n + 512, X + 8))[what]
    result = [n, said(dev.attn_paged_dev, c, b, attn(workspace=at, workspace_bytes=size))]
""")
    assert got[0] > 0
    if what == "exact":
        assert got[1] == ""
    elif what == "capture":
        assert "capture" in got[1] and got[2] == ""
    else:
        assert "workspace" in got[1]


@pytest.mark.parametrize("call,want", [
    # single tokens: blocks of 16 rows, a wave each where they fill the device
    ("batch(), attn()", ["attnp_rows_kernel<2,4,4>"]),
    ("batch(n_req=200, n_tok=200), attn()", ["attnp_rows_kernel<2,4,1>"]),
    ("batch(n_req=300, n_tok=300), attn()", ["attnp_rows_kernel<2,4,4>"]),
    # prompts: large blocks from some work on, split and joined where they are few
    ("batch(n_req=1, n_tok=200, max_q=200), attn()", ["attnp_rows_kernel<2,4,4>"]),
    ("batch(n_req=1, n_tok=1500, max_q=1500, max_kv=1500), attn()", ["attnp_rows_kernel<2,4,1>"]),
    ("batch(n_req=1, n_tok=4096, max_q=4096, max_kv=4096), attn()", ["attnp_tiles_kernel<8,8>"]),
    ("batch(n_req=1, n_tok=512, max_q=512, max_kv=4512), attn()", ["attnp_tiles_kernel<8,8>", "attnp_join_kernel<256>"]),
    # beside single tokens, which have their own launch
    ("batch(n_req=9, n_tok=4104, max_q=4096, max_kv=4096), attn()", ["attnp_rows_kernel<2,4,4>", "attnp_tiles_kernel<8,8>"]),
    # other heads
    ("batch(n_req=1, n_tok=4096, max_q=4096, max_kv=4096), attn()|head_dim=64", ["attnp_tiles_kernel<4,4>"]),
    ("batch(n_req=1, n_tok=4096, max_q=4096, max_kv=4096), attn()|head_dim=96", ["attnp_tiles_kernel<6,8>"]),
    ("batch(n_req=1, n_tok=4096, max_q=4096, max_kv=4096), attn(ldq=8192, ldo=8192)|head_dim=256", ["attnp_rows_kernel<4,2,1>"]),
    ("batch(), attn(ldq=8192, ldo=8192)|head_dim=144", ["attnp_rows_kernel<3,2,4>"]),
    ("batch(), attn()|head_dim=16", ["attnp_rows_kernel<1,4,4>"])])
def test_the_kernels_of_a_shape(call, want):
    args, _, heads = call.partition("|")
    got = fake_hip.run(SETUP + f"batch_ = batch\ndef batch(**o): return batch_(max_blocks=200, **o)\ndev.attn_paged_dev(cache({heads}), {args}); result = launched()")
    assert sorted(k for k, *_ in got) == sorted(want)


@pytest.mark.parametrize("block,hd,want", [(16, 64, "1,128"), (16, 128, "1,128"), (32, 128, "1,256"), (64, 128, "1,512"),
                                           (128, 128, "1,1024"), (256, 128, "2,1024"), (256, 256, "4,1024")])
def test_the_kernels_of_a_page(block, hd, want):
    got = fake_hip.run(SETUP + f"""
c = cache(block={block}, head_dim={hd})
dev.kv_append_dev(c, batch(), X, 4096, X, 4096)
for n in 600, 5000:
    dev.kv_read_dev(c, X, n, X, 4096, X, 4096)
dev.kv_plan_dev(plan(n_req=256))
dev.kv_plan_dev(plan(n_req=257))
result = launched()
""")
    assert [k for k, *_ in got] == [f"kv_append_kernel<{want}>", "kv_read_kernel<16>", "kv_read_kernel<64>", "kv_plan_kernel<256>",
                                    "kv_plan_kernel<1024>"]


def test_as_many_pieces_as_counters():
    """Many requests over splits that an option asks for: more pieces than
    the workspace has counters are not made."""
    got = fake_hip.run(SETUP + """
dev.set_option("ATTNP_SPLITS", 64)
c, a = cache(n_pages=1 << 20), attn()
big, few = (batch(n_req=n, n_tok=n, max_blocks=200, max_kv=6400) for n in (4096, 100))
result = [dev.attn_paged_workspace(c, b, a) for b in (big, few)]
dev.attn_paged_dev(c, big, a)
result.append(launched())
""")
    assert got[0] == 0 and got[1] > 0 and got[2] == [["attnp_rows_kernel<2,4,4>", 1, 8]]


def test_a_failed_launch_is_reported():
    for call in ("kv_plan_dev(plan())", "kv_append_dev(cache(), batch(), X, 4096, X, 4096)",
                 "kv_read_dev(cache(), X, 4, X, 4096, X, 4096)", "attn_paged_dev(cache(), batch(), attn())"):
        got = fake_hip.run(SETUP + f"""
fake.fake_reset(1)
try:
    dev.{call}
    result = ""
except sa.SihipError as e:
    result = str(e)
""")
        assert "error -8" in got, call
