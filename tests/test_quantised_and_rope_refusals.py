"""What the preparation of ragged rows and the quantised cache refuse before any launch, the
frequencies of rotary positions and the plan of the quantised decode. Runs without a GPU:
no call here reaches the device."""
import ctypes
import math
import subprocess
from pathlib import Path

import numpy as np
import pytest

import gemma_kv as gk

OK = 0
BAD = gk.HIP_ERROR_INVALID_VALUE
P = 0x100000  # an aligned address that nobody reads


def cfg(layers=2, pages=64, page=16, max_pages=16, batch=4, heads=8, dim=256, window=0):
    return gk.make_config(layers, pages, page, max_pages, batch, heads, dim, window)


# ---- frequencies ---------------------------------------------------------------------

def frequencies(**change):
    a = dict(turns=np.zeros(256), amplitude=gk._F32(), rotary=128, exponent=128, theta=1e4, scaling=0, factor=1.0,
             context=0.0, fast=32.0, slow=1.0)
    a.update(change)
    turns = a["turns"]
    return gk.lib().gemma4_rope_frequencies(
        turns.ctypes.data if turns is not None else None,
        ctypes.byref(a["amplitude"]) if a["amplitude"] is not None else None, a["rotary"], a["exponent"], a["theta"],
        a["scaling"], a["factor"], a["context"], a["fast"], a["slow"])


@pytest.mark.parametrize("what", [
    dict(turns=None), dict(amplitude=None), dict(rotary=0), dict(rotary=-2), dict(rotary=7), dict(rotary=514, exponent=514),
    dict(rotary=256), dict(theta=1.0), dict(theta=-1e4), dict(theta=float("nan")), dict(theta=float("inf")),
    dict(scaling=-1), dict(scaling=4), dict(scaling=1, factor=0.5), dict(scaling=1, factor=float("nan")),
    dict(scaling=2, factor=float("inf")), dict(scaling=2, rotary=2, exponent=2, factor=2.0),
    dict(scaling=3, factor=2.0, context=0.0), dict(scaling=3, factor=2.0, context=4096.0, fast=1.0),
    dict(scaling=3, factor=2.0, context=4096.0, slow=-1.0), dict(scaling=3, factor=2.0, context=float("nan")),
    dict(scaling=3, factor=2.0, context=4096.0, fast=float("inf"))])
def test_frequencies_refuse(what):
    assert frequencies(**what) == BAD


def test_frequencies_take_what_a_kind_does_not_name():
    assert frequencies(factor=0.0, context=-1.0, fast=0.0, slow=float("nan")) == OK
    assert frequencies(scaling=1, factor=4.0, context=-1.0, fast=0.0) == OK


@pytest.mark.parametrize("rotary,exponent", [(256, 256), (128, 512), (16, 16), (512, 512)])
@pytest.mark.parametrize("theta", [1e4, 1e6])
def test_frequencies(rotary, exponent, theta):
    """A few roundings of 64 bits, of the logarithm's size: 2^-46 of a frequency."""
    i = np.arange(rotary // 2)
    plain = theta ** (-2 * i / exponent) / (2 * math.pi)
    near = dict(rtol=2.0**-46, atol=0)
    get = lambda *a, **k: gk.rope_frequencies(rotary, theta, *a, exponent_dim=exponent, **k)  # noqa: E731
    turns, amplitude = get()
    assert amplitude == 1.0
    np.testing.assert_allclose(turns, plain, **near)
    turns, amplitude = get(gk.ROPE_LINEAR, 8.0)
    assert amplitude == 1.0
    np.testing.assert_allclose(turns, plain / 8, **near)
    turns, amplitude = get(gk.ROPE_BASE, 8.0)
    assert amplitude == 1.0
    np.testing.assert_allclose(turns, (theta * 8 ** (exponent / (exponent - 2))) ** (-2 * i / exponent) / (2 * math.pi), **near)
    assert turns[0] == get()[0][0]
    turns, amplitude = get(gk.ROPE_BY_PARTS, 8.0, 4096.0)
    kept = np.clip((plain * 4096 - 1) / 31, 0, 1)
    np.testing.assert_allclose(turns, plain * kept + plain * (1 - kept) / 8, rtol=2.0**-40)
    assert amplitude == np.float32(0.1 * math.log(8) + 1)
    assert turns[0] == plain[0] if plain[0] * 4096 > 32 else True
    turns, amplitude = get(gk.ROPE_BY_PARTS, 1.0, 4096.0)
    np.testing.assert_allclose(turns, plain, **near)
    assert amplitude == 1.0


# ---- rows ----------------------------------------------------------------------------

def rope(**change):
    a = dict(q_out=P, k_out=P, v_out=P, q=P, k=P, v=P, wq=P, wk=P, position=P, turns=P, amplitude=1.0, rotary=64,
             interleaved=False, heads=8, dim=256, rows=3, q_stride=0, kv_stride=0)
    a.update(change)
    return gk.rope_rows_bf16(a["q_out"], a["k_out"], a["v_out"], a["q"], a["k"], a["v"], a["wq"], a["wk"], a["position"],
                             a["turns"], a["amplitude"], a["rotary"], a["interleaved"], a["heads"], a["dim"], a["rows"],
                             stream=0, q_stride=a["q_stride"], kv_stride=a["kv_stride"])


@pytest.mark.parametrize("what", [
    *[{n: 0} for n in ("q_out", "k_out", "q", "k", "position", "turns", "v_out")],
    *[{n: P + 8} for n in ("q_out", "k_out", "v_out", "q", "k", "v", "wq", "wk")], dict(turns=P + 4),
    dict(rows=-1), dict(rows=(1 << 22) + 1), dict(rotary=0), dict(rotary=8), dict(rotary=72), dict(rotary=272),
    dict(heads=1, dim=512, rotary=528), dict(heads=1), dict(dim=512), dict(heads=16), dict(heads=4, dim=128),
    dict(amplitude=float("nan")), dict(amplitude=float("inf")), dict(q_stride=4088), dict(q_stride=4100),
    dict(kv_stride=2040), dict(kv_stride=2052), dict(q_stride=(1 << 30) + 8), dict(kv_stride=(1 << 30) + 8),
    dict(q_stride=-4096)])
def test_rows_refuse(what):
    assert rope(**what) == BAD


def test_no_rows():
    assert rope(rows=0, q=0) == OK


def fp8_rows(call, **change):
    a = dict(ck=P, cv=P, config=cfg(), table=P, tb=P, tp=P, n=5, layer=0, k=P, v=P, ks=P, vs=P, kv_stride=0)
    a.update(change)
    cache, rows, tokens = (a["ck"], a["cv"]), (a["k"], a["v"]), (a["config"], a["table"], a["tb"], a["tp"], a["n"], a["layer"])
    if call == "write":
        return gk.kv_cache_write_fp8(*cache, *tokens, *rows, a["ks"], a["vs"], stream=0, kv_stride=a["kv_stride"])
    return gk.kv_cache_read_fp8(*rows, *cache, *tokens, a["ks"], a["vs"], stream=0, kv_stride=a["kv_stride"])


@pytest.mark.parametrize("call", ["write", "read"])
@pytest.mark.parametrize("what", [
    *[{n: 0} for n in ("ck", "cv", "table", "tb", "tp", "k", "v")], *[{n: P + 8} for n in ("ck", "cv", "k", "v")],
    dict(n=-1), dict(layer=-1), dict(layer=2), dict(config=cfg(page=0)), dict(config=cfg(pages=0)),
    dict(config=cfg(max_pages=0)), dict(config=cfg(batch=0)), dict(config=cfg(heads=0)), dict(config=cfg(dim=0)),
    dict(config=cfg(dim=24)), dict(config=cfg(window=-1)), dict(config=cfg(heads=4096, dim=512)),
    dict(kv_stride=2040), dict(kv_stride=2052), dict(kv_stride=(1 << 30) + 8), dict(kv_stride=-2048),
    dict(n=2**31 - 1)])
def test_quantised_rows_refuse(call, what):
    assert fp8_rows(call, **what) == BAD


def test_no_quantised_rows():
    assert fp8_rows("write", n=0, k=0) == OK and fp8_rows("read", n=0, k=0) == OK


# ---- attention over codes ------------------------------------------------------------

def decode(append, **change):
    a = dict(out=P, m=P, l=P, acc=P, q=P, ck=P, cv=P, ks=P, vs=P, table=P, lengths=P, position=P, k=P, v=P, config=cfg(),
             layer=0, scale=0.0625, size=32, splits=4, batch=4)
    a.update(change)
    head = [a[n] for n in ("out", "m", "l", "acc", "q", "ck", "cv", "ks", "vs", "table", "lengths")]
    tail = [a[n] for n in ("config", "layer", "scale", "size", "splits", "batch")]
    if append:
        return gk.flash_attention_append_decode_paged_fp8(*head, a["position"], a["k"], a["v"], *tail, stream=0)
    return gk.flash_attention_decode_paged_fp8(*head, *tail, stream=0)


@pytest.mark.parametrize("append", [False, True])
@pytest.mark.parametrize("what", [
    *[{n: 0} for n in ("out", "m", "l", "acc", "q", "ck", "cv", "table", "lengths")],
    *[{n: P + 8} for n in ("out", "acc", "q", "ck", "cv")],
    dict(layer=-1), dict(layer=2), dict(batch=-1), dict(batch=5), dict(size=0), dict(size=-32), dict(splits=0),
    dict(splits=65536), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")),
    dict(config=cfg(heads=1)), dict(config=cfg(dim=512)), dict(config=cfg(heads=4, dim=512)),
    dict(config=cfg(window=1024)), dict(config=cfg(pages=1 << 24, page=64, layers=2)), dict(config=cfg(page=0))])
def test_attention_over_codes_refuses(append, what):
    assert decode(append, **what) == BAD


@pytest.mark.parametrize("what", [{n: 0} for n in ("position", "k", "v")] + [{n: P + 8} for n in ("k", "v")])
def test_append_over_codes_refuses(what):
    assert decode(True, **what) == BAD


def test_no_sequences():
    assert decode(False, batch=0, q=0) == OK and decode(True, batch=0, q=0) == OK


@pytest.mark.parametrize("heads,dim", [(8, 256), (1, 512)])
def test_plan_covers_the_keys(heads, dim):
    c = cfg(heads=heads, dim=dim)
    for batch in (1, 2, 7, 64, 4096):
        for keys in (0, 1, 31, 32, 33, 1024, 8193, 131072, 2**31 - 1):
            size, splits = gk.decode_split_plan_fp8(c, batch, keys)
            assert size > 0 and splits > 0 and size * splits >= keys and size * (splits - 1) < max(keys, 1)
            assert splits <= 65535 and size % 32 == 0
    assert gk.decode_split_plan_fp8(c, 1, 4096, 8 if heads == 8 else 1)[1] == 1


@pytest.mark.parametrize("change", [dict(heads=4), dict(dim=128), dict(heads=8, dim=512)])
def test_plan_refuses(change):
    with pytest.raises(gk.HipError):
        gk.decode_split_plan_fp8(cfg(**change), 1, 100)
    with pytest.raises(gk.HipError):
        gk.decode_split_plan_fp8(cfg(), 0, 100)
    with pytest.raises(gk.HipError):
        gk.decode_split_plan_fp8(cfg(), 1, -1)


# ---- groups that share a prefix --------------------------------------------------------

def shared_plan(config=None, batch=4, rows=10, groups=1, plan_ptr=P, offsets=P, prior=P, table=P, at=P, nbytes=None):
    config = config or cfg()
    n = gk.flash_attention_extend_shared_plan_bytes(config, batch, rows) if nbytes is None else nbytes
    return gk.flash_attention_extend_shared_plan(plan_ptr, n, offsets, prior, table, at, groups, config, batch, rows, 0)


@pytest.mark.parametrize("what", [
    dict(config=cfg(heads=8, dim=512)), dict(config=cfg(heads=4)), dict(batch=0), dict(batch=5), dict(rows=-1),
    dict(rows=(1 << 24) + 1), dict(config=cfg(batch=5000), batch=4097), dict(config=cfg(page=0)),
    dict(config=cfg(window=64)), dict(groups=-1), dict(groups=2049), dict(plan_ptr=0), dict(plan_ptr=P + 128),
    dict(offsets=0), dict(prior=0), dict(table=0), dict(at=0), dict(nbytes=255)])
def test_shared_plan_refuses(what):
    assert shared_plan(**what) == BAD


def test_shared_plan_needs_its_bytes():
    n = gk.flash_attention_extend_shared_plan_bytes(cfg(), 4, 10)
    assert shared_plan(nbytes=n - 1) == BAD
    assert gk.flash_attention_extend_shared_plan_bytes(cfg(window=64), 4, 10) == 0
    assert gk.flash_attention_extend_shared_workspace_bytes(cfg(window=64), 4, 10) == 0
    assert gk.flash_attention_extend_shared_plan_bytes(cfg(), 0, 10) == 0
    assert n > gk.flash_attention_extend_plan_bytes(cfg(), 4, 10)
    for heads, dim in ((8, 256), (1, 512)):
        c = cfg(heads=heads, dim=dim, batch=4096)
        last = (0, 0)
        for rows in (0, 1, 2, 63, 64, 65, 96, 97, 128, 1000, 1 << 16, 1 << 24):
            size = (gk.flash_attention_extend_shared_workspace_bytes(c, 64, rows),
                    gk.flash_attention_extend_shared_plan_bytes(c, 64, rows))
            assert size[0] >= last[0] and size[1] >= last[1] and size[1] > 0
            last = size


def shared_attend(**change):
    config = change.pop("config", None) or cfg()
    rows, batch = change.pop("rows", 10), change.pop("batch", 4)
    a = dict(out=P, q=P, k=P, v=P, cache_k=P, cache_v=P, page_table=P, plan=P,
             plan_bytes=gk.flash_attention_extend_shared_plan_bytes(config, batch, rows), config=config, layer=0,
             batch_size=batch, total_rows=rows, softmax_scale=0.0625, workspace=P,
             workspace_bytes=gk.flash_attention_extend_shared_workspace_bytes(config, batch, rows), stream=0,
             q_stride=0, kv_stride=0)
    a.update(change)
    return gk.flash_attention_extend_shared_paged_bf16(**a)


@pytest.mark.parametrize("what", [
    *[{n: 0} for n in ("out", "q", "k", "v", "cache_k", "cache_v", "page_table", "plan", "workspace")],
    *[{n: P + 8} for n in ("out", "q", "k", "v", "cache_k", "cache_v")],
    dict(plan=P + 16), dict(workspace=P + 16), dict(layer=-1), dict(layer=2), dict(batch_size=0), dict(batch_size=5),
    dict(total_rows=-1), dict(softmax_scale=0.0), dict(softmax_scale=float("nan")), dict(q_stride=4088),
    dict(q_stride=4100), dict(kv_stride=2040), dict(kv_stride=(1 << 30) + 8), dict(plan_bytes=1), dict(workspace_bytes=1),
    dict(config=cfg(window=64))])
def test_shared_attention_refuses(what):
    assert shared_attend(**what) == BAD


def test_shared_attention_without_rows():
    assert shared_attend(rows=0, q=0) == OK


def test_c_caller(tmp_path):
    """The same interface from plain C, compiled with gcc against the headers."""
    repo = Path(__file__).resolve().parent.parent
    lib = repo / "gemma.c_amd" / "gemma_kv"
    exe = tmp_path / "quantised_caller"
    cmd = ["gcc", "-std=c11", "-Wall", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include", f"-I{repo / 'include'}",
           str(repo / "tests" / "cpp" / "quantised_caller.c"), f"-L{lib}", "-lgemma4_kv", f"-Wl,-rpath,{lib}",
           "-o", str(exe)]
    proc = subprocess.run(cmd, capture_output=True, text=True, timeout=300)
    assert proc.returncode == 0, proc.stderr
    assert "quantised caller ok" in subprocess.run([str(exe)], capture_output=True, text=True, timeout=60).stdout
