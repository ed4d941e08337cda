"""What the ragged extension attention and the page pool refuse before any
launch: bad sizes, null and misaligned pointers, windows that a cache cannot
hold. Runs without a GPU: no call here reaches the device."""
import subprocess
from pathlib import Path

import pytest

import gemma_kv as gk

OK = 0
BAD = gk.HIP_ERROR_INVALID_VALUE
P = 0x100000  # an aligned address that nobody reads


def cfg(layers=2, pages=64, page=16, max_pages=16, batch=4, heads=8, dim=256, window=0):
    return gk.make_config(layers, pages, page, max_pages, batch, heads, dim, window)


RING = dict(window=64, max_pages=8, pages=32)


def plan(config=None, batch=4, rows=10, window=0, sinks=0, plan_ptr=P, offsets=P, prior=P, nbytes=None):
    config = config or cfg()
    n = gk.flash_attention_extend_plan_bytes(config, batch, rows) if nbytes is None else nbytes
    return gk.flash_attention_extend_plan(plan_ptr, n, offsets, prior, config, batch, rows, window, sinks, 0)


@pytest.mark.parametrize("what", [
    dict(config=cfg(heads=8, dim=512)), dict(config=cfg(heads=1, dim=256)), dict(config=cfg(heads=4)),
    dict(batch=0), dict(batch=-1), dict(batch=5), dict(rows=-1), dict(rows=(1 << 24) + 1),
    dict(config=cfg(batch=5000), batch=4097), dict(config=cfg(page=0)), dict(config=cfg(pages=0)),
    dict(config=cfg(max_pages=0)), dict(config=cfg(layers=0)), dict(window=-1), dict(sinks=-1),
    dict(plan_ptr=0), dict(plan_ptr=P + 128), dict(offsets=0), dict(prior=0), dict(nbytes=255),
    # A ring: a window of its own size at most, that it has the slots for, and no sinks.
    dict(config=cfg(**RING), window=0), dict(config=cfg(**RING), window=65),
    dict(config=cfg(**RING), window=64, sinks=1),
    dict(config=cfg(window=256, max_pages=8, pages=32), window=129)])
def test_plan_refuses(what):
    assert plan(**what) == BAD


def attend(**change):
    config = change.pop("config", None) or cfg()
    rows, batch = change.pop("rows", 10), change.pop("batch", 4)
    a = dict(out=P, q=P, k=P, v=P, cache_k=P, cache_v=P, page_table=P, plan=P,
             plan_bytes=gk.flash_attention_extend_plan_bytes(config, batch, rows), config=config, layer=0,
             batch_size=batch, total_rows=rows, softmax_scale=0.0625, workspace=P,
             workspace_bytes=gk.flash_attention_extend_workspace_bytes(config, batch, rows), stream=0,
             q_stride=0, kv_stride=0)
    a.update(change)
    return gk.flash_attention_extend_paged_bf16(**a)


@pytest.mark.parametrize("what", [
    *[{n: 0} for n in ("out", "q", "k", "v", "cache_k", "cache_v", "page_table", "plan", "workspace")],
    *[{n: P + 8} for n in ("out", "q", "k", "v", "cache_k", "cache_v")],
    dict(plan=P + 16), dict(workspace=P + 16), dict(layer=-1), dict(layer=2), dict(batch_size=0),
    dict(batch_size=5), dict(total_rows=-1), dict(softmax_scale=0.0), dict(softmax_scale=-1.0),
    dict(softmax_scale=float("nan")), dict(softmax_scale=float("inf")), dict(q_stride=4088),
    dict(q_stride=4100), dict(kv_stride=2040), dict(kv_stride=2052), dict(q_stride=-4096),
    dict(kv_stride=1 << 32), dict(plan_bytes=255), dict(workspace_bytes=255),
    dict(config=cfg(heads=2, dim=256))])
def test_attention_refuses(what):
    assert attend(**what) == BAD


def test_no_rows_is_a_success():
    assert attend(rows=0) == OK


def test_sizes():
    """A larger call's buffers hold a smaller one's; a bad configuration has no size."""
    for heads, dim in ((8, 256), (1, 512)):
        c = cfg(batch=64, heads=heads, dim=dim)
        for size in (gk.flash_attention_extend_plan_bytes, gk.flash_attention_extend_workspace_bytes):
            most = size(c, 64, 5000)
            for batch in (1, 2, 63, 64):
                for rows in (0, 1, 2, 7, 8, 9, 63, 64, 65, 1000, 5000):
                    assert 0 < size(c, batch, rows) <= most or rows == 0
            assert size(cfg(heads=3), 1, 1) == 0 and size(c, 65, 1) == 0


POOL_BAD = [dict(config=cfg(pages=0)), dict(config=cfg(page=0)), dict(config=cfg(max_pages=0)),
            dict(config=cfg(batch=0)), dict(config=cfg(batch=4097)), dict(config=cfg(window=-1)),
            dict(config=cfg(batch=4096, max_pages=1 << 20)), dict(config=cfg(pages=1 << 20, page=1 << 12))]


def reserve(**change):
    a = dict(page_table=P, page_refs=P, config=cfg(), first_position=P, end_position=P, status=P, stream=0)
    a.update(change)
    return gk.kv_cache_reserve_pages(**a)


@pytest.mark.parametrize("what", POOL_BAD + [{n: 0} for n in (
    "page_table", "page_refs", "first_position", "end_position", "status")])
def test_reserve_refuses(what):
    assert reserve(**what) == BAD


@pytest.mark.parametrize("what", POOL_BAD + [{n: 0} for n in (
    "page_table", "page_refs", "first_position", "end_position")])
def test_release_refuses(what):
    a = dict(page_table=P, page_refs=P, config=cfg(), first_position=P, end_position=P, stream=0)
    a.update(what)
    assert gk.kv_cache_release_pages(**a) == BAD


ROWS_BAD = [dict(config=cfg(layers=0)), dict(config=cfg(heads=0)), dict(config=cfg(dim=0)), dict(config=cfg(dim=12)),
            dict(cache_k=0), dict(cache_v=0), dict(cache_k=P + 8), dict(cache_v=P + 8)]


def fork(**change):
    a = dict(cache_k=P, cache_v=P, config=cfg(), page_table=P, page_refs=P, seq_lengths=P, parents=P, children=P,
             fork_count=2, status=P, stream=0)
    a.update(change)
    return gk.kv_cache_fork_bf16(**a)


@pytest.mark.parametrize("what", POOL_BAD + ROWS_BAD + [dict(fork_count=-1), dict(fork_count=5)] + [{n: 0} for n in (
    "page_table", "page_refs", "seq_lengths", "parents", "children", "status")])
def test_fork_refuses(what):
    assert fork(**what) == BAD


def compact(**change):
    a = dict(cache_k=P, cache_v=P, config=cfg(), page_table=P, page_refs=None, sequences=P, first_positions=P,
             kept_offsets=P, kept_positions=P, sequence_count=2, total_kept=5, status=P, stream=0)
    a.update(change)
    return gk.kv_cache_compact_bf16(**a)


@pytest.mark.parametrize("what", POOL_BAD + ROWS_BAD + [
    dict(sequence_count=-1), dict(sequence_count=5), dict(total_kept=-1)] + [{n: 0} for n in (
        "page_table", "sequences", "first_positions", "kept_offsets", "kept_positions", "status")])
def test_compact_refuses(what):
    assert compact(**what) == BAD


def test_nothing_to_do_is_a_success():
    assert fork(fork_count=0) == OK and compact(sequence_count=0) == OK


def test_c_caller(tmp_path):
    """The same interface from plain C, compiled with gcc against the headers."""
    repo = Path(__file__).resolve().parent.parent
    lib = repo / "gemma.c_amd" / "gemma_kv"
    exe = tmp_path / "serving_caller"
    cmd = ["gcc", "-std=c11", "-Wall", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include", f"-I{repo / 'include'}",
           str(repo / "tests" / "cpp" / "serving_caller.c"), f"-L{lib}", "-lgemma4_kv", f"-Wl,-rpath,{lib}",
           "-o", str(exe)]
    proc = subprocess.run(cmd, capture_output=True, text=True, timeout=300)
    assert proc.returncode == 0, proc.stderr
    assert "serving caller ok" in subprocess.run([str(exe)], capture_output=True, text=True, timeout=60).stdout


@pytest.mark.parametrize("config", [
    cfg(batch=4096, page=1024, max_pages=64, pages=4096, window=60000),  # a ring: every page may be copied
    cfg(batch=4096, page=1 << 19, max_pages=2, pages=64)])               # a begun page of 2^19 rows each
def test_fork_refuses_more_copies_than_a_launch_holds(config):
    """Before the tables' launch, which could not be taken back."""
    assert fork(config=config, fork_count=4096) == BAD
