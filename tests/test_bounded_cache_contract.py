"""The bounded-cache launchers' refusals and host arithmetic, through the C ABI without a device: every call here is
answered before anything is launched."""
import ctypes as C
import time

import pytest

from redline_llm_b200 import kernels as K

NULL, SHAPE, WORKSPACE, LARGE = -1, -2, -3, -4
P = 4096          # a stand-in pointer: aligned, never dereferenced by a refused call


def decode(**kw):
    a = dict(out=P, os=1536, q=P, qs=2048, pool=P, tab=P, lens=P, n=4, mb=8, qh=12, kvh=2, d=128, scale=0.1, window=64,
             sinks=4, ws=P, wb=1 << 40)
    a.update(kw)
    return K.lib().rl_launch_paged_window_attention_decode(a["out"], a["os"], a["q"], a["qs"], a["pool"], a["tab"],
                                                           a["lens"], a["n"], a["mb"], a["qh"], a["kvh"], a["d"],
                                                           a["scale"], a["window"], a["sinks"], a["ws"], a["wb"], None)


def weights(**kw):
    a = dict(out=P, os=1536, q=P, qs=2048, pool=P, tab=P, lens=P, n=4, mb=8, qh=12, kvh=2, d=128, scale=0.1, w=P, ws=P,
             wb=1 << 40)
    a.update(kw)
    return K.lib().rl_launch_paged_attention_decode_weights(a["out"], a["os"], a["q"], a["qs"], a["pool"], a["tab"],
                                                            a["lens"], a["n"], a["mb"], a["qh"], a["kvh"], a["d"],
                                                            a["scale"], a["w"], a["ws"], a["wb"], None)


def prefill(**kw):
    a = dict(out=P, os=1536, q=P, qs=2048, pool=P, tab=P, mb=8, start=0, n=100, qh=12, kvh=2, d=128, scale=0.1,
             window=64, sinks=4, ws=None, wb=0)
    a.update(kw)
    return K.lib().rl_launch_paged_window_prefill_attention(a["out"], a["os"], a["q"], a["qs"], a["pool"], a["tab"],
                                                            a["mb"], a["start"], a["n"], a["qh"], a["kvh"], a["d"],
                                                            a["scale"], a["window"], a["sinks"], a["ws"], a["wb"], None)


def evict(**kw):
    a = dict(pool=P, w=P, tab=P, mb=8, dst=2 * P, dmb=4, lens=P, new=P, kept=P, n=4, kvh=2, d=128, budget=64, sinks=4,
             recent=16)
    a.update(kw)
    return K.lib().rl_launch_kv_evict(a["pool"], a["w"], a["tab"], a["mb"], a["dst"], a["dmb"], a["lens"], a["new"],
                                      a["kept"], a["n"], a["kvh"], a["d"], a["budget"], a["sinks"], a["recent"], None)


ATTENTION_SHAPES = [dict(d=64), dict(d=256), dict(kvh=0), dict(kvh=9, qh=9, os=9 * 128, qs=9 * 128), dict(kvh=-1),
                    dict(qh=13), dict(qh=1), dict(qh=18, os=18 * 128, qs=18 * 128), dict(mb=0), dict(mb=-5), dict(os=1535),
                    dict(qs=1000), dict(scale=0.0), dict(scale=-0.1), dict(scale=float("nan")),
                    dict(scale=float("inf")), dict(scale=3.0e38), dict(pool=P + 8)]


@pytest.mark.parametrize("call", [decode, weights, prefill])
@pytest.mark.parametrize("change", ATTENTION_SHAPES)
def test_shapes_the_attention_launchers_refuse(call, change):
    if call is prefill and change.get("mb") in (0, -5):
        change = dict(change, n=1)
    assert call(**change) == SHAPE
    assert K.lib().rl_last_error()


@pytest.mark.parametrize("call", [decode, weights, prefill])
@pytest.mark.parametrize("name", ["out", "q", "pool", "tab"])
def test_null_pointers_are_refused(call, name):
    assert call(**{name: None}) == NULL


def test_refusals_of_one_launcher_only():
    for call in (decode, weights):
        assert call(lens=None) == NULL and call(ws=None) == NULL
        assert call(qs=2047) == SHAPE and call(q=P + 2) == SHAPE and call(ws=P + 8) == SHAPE
        assert call(mb=(1 << 26) + 1) == LARGE
        assert call(wb=0) == WORKSPACE
        assert call(**dict(dict(mb=1 << 26, n=64, wb=(1 << 64) - 1), **(dict(window=2**31 - 1) if call is decode else {}))) == LARGE
        need = K.window_attention_workspace_bytes(4, 8, 12, 2, weights=call is weights)
        assert call(wb=need - 1) == WORKSPACE and b"workspace" in K.lib().rl_last_error()
        assert call(n=0, out=None) == 0 and call(n=-3, out=None) == 0
    assert weights(w=None) == NULL and weights(w=P + 2) == SHAPE
    for call in (decode, prefill):
        assert call(window=0) == SHAPE and call(window=-1) == SHAPE and call(sinks=-1) == SHAPE
    assert prefill(n=0, out=None) == 0
    assert prefill(start=-1) == SHAPE and prefill(n=129) == SHAPE and prefill(start=29) == SHAPE
    assert prefill(start=2**31 - 1, n=2**31 - 1) == SHAPE
    assert prefill(q=P + 8) == SHAPE and prefill(out=P + 8) == SHAPE and prefill(qs=2044) == SHAPE
    assert prefill(os=1540) == SHAPE


def test_evict_refusals():
    for name in ("pool", "w", "tab", "dst", "lens", "new", "kept"):
        assert evict(**{name: None}) == NULL
    for change in (dict(kvh=0), dict(kvh=65536), dict(d=0), dict(d=4), dict(d=100), dict(d=1032), dict(mb=0), dict(dmb=0),
                   dict(budget=0), dict(budget=-1), dict(sinks=-1), dict(recent=-1), dict(sinks=60, recent=5),
                   dict(sinks=2**31 - 1, recent=2**31 - 1), dict(budget=65), dict(dst=P), dict(pool=P + 8), dict(w=P + 2)):
        assert evict(**change) == SHAPE, change
    assert evict(budget=(1 << 30) + 1, mb=1 << 26, dmb=1 << 26) == LARGE and evict(n=1 << 28) == LARGE
    assert evict(mb=(1 << 26) + 1) == LARGE and evict(dmb=(1 << 26) + 1) == LARGE
    assert evict(n=0, pool=None) == 0 and evict(n=-1, pool=None) == 0


def test_workspace_queries():
    size = K.window_attention_workspace_bytes
    assert 0 < size(1, 1, 1, 1) <= size(64, 1, 12, 2) <= size(64, 2048, 12, 2)
    assert size(64, 2048, 12, 2, weights=True) >= size(64, 2048, 12, 2)
    assert size(8, 100, 12, 2, weights=True) <= size(9, 100, 12, 2, weights=True) <= size(9, 101, 12, 2, weights=True)
    assert size(0, 1, 12, 2) >= 0
    for bad in ((-1, 1, 12, 2), (1, 0, 12, 2), (1, 1, 12, 9), (1, 1, 12, 0), (1, 1, 18, 2), (1, 1, 7, 2)):
        with pytest.raises(K.KernelError):
            size(*bad)
    out = C.c_size_t(7)
    L = K.lib()
    for bad in ((-1, 1, 12, 1, 0), (0, -1, 12, 1, 0), (0, 1, 0, 1, 0), (0, 1, 12, 0, 0), (0, 1, 12, 1, -1)):
        assert L.rl_window_prefill_workspace_bytes(*bad, C.byref(out)) == SHAPE and out.value == 0
    assert L.rl_window_prefill_workspace_bytes(0, 1, 12, 1, 0, None) == NULL
    assert L.rl_window_attention_workspace_bytes(1, 1, 12, 2, 0, None) == NULL
    assert L.rl_window_attention_health(None, None) == NULL


def test_arrays_that_would_be_written_past_their_end_are_refused():
    """By the Python wrappers, before anything else is looked at."""
    torch = pytest.importorskip("torch")
    t = torch.zeros(4, 8, dtype=torch.int32)
    lens, w, kept = torch.zeros(4, dtype=torch.int32), torch.zeros(9, 2, 16), torch.zeros(4, 2, 64, dtype=torch.int32)

    def evict(w=w, new=lens, kept=kept):
        K.launch_kv_evict(t, w, t, 8, t, 8, lens, new, kept, 4, 2, 128, 64, 4, 16)

    for bad in (dict(w=w.half()), dict(w=w.double()), dict(w=torch.zeros(9, 2, 32)[:, :, ::2]), dict(kept=kept.short()),
                dict(kept=kept[:3]), dict(kept=kept[:, :1].expand(4, 2, 64)), dict(new=lens.long()), dict(new=lens[:3])):
        with pytest.raises(K.KernelError, match="must be a contiguous"):
            evict(**bad)
    with pytest.raises(K.KernelError, match="must be a contiguous"):
        K.launch_paged_attention_decode_weights(t, 1536, t, 1536, t, t, lens, 4, 8, 12, 2, 128, 0.1, w.half(), t)


def test_weights_must_cover_the_pool_and_tables_and_lengths_be_int32():
    """The kernels address weights, tables and lengths by the pool's page numbers and the call's counts: an array with fewer
    pages than the pool would be written past its end, 64-bit tables read as pairs of wrong page numbers. Refused by the
    wrappers for every layout of the pool tensor, before a device is looked at."""
    torch = pytest.importorskip("torch")
    blocks, kv, d, rows, mb = 9, 2, 128, 4, 8
    pool = torch.zeros(blocks, 2, kv, 16, d, dtype=torch.float16)
    good = dict(w=torch.zeros(blocks, kv, 16), tab=torch.zeros(rows, mb, dtype=torch.int32),
                dst=torch.zeros(rows, 4, dtype=torch.int32), lens=torch.zeros(rows, dtype=torch.int32),
                out=torch.zeros(rows, 12 * d, dtype=torch.float16), pool=pool)
    new, kept = torch.zeros(rows, dtype=torch.int32), torch.zeros(rows, kv, 64, dtype=torch.int32)
    ws, q = torch.zeros(1 << 20, dtype=torch.uint8), torch.zeros(rows, 12 * d, dtype=torch.float16)

    def evict(**kw):
        a = dict(good, **kw)
        K.launch_kv_evict(a["pool"], a["w"], a["tab"], mb, a["dst"], 4, a["lens"], new, kept, rows, kv, d, 64, 4, 16)

    def weights(**kw):
        a = dict(good, **kw)
        K.launch_paged_attention_decode_weights(a["out"], 12 * d, q, 12 * d, a["pool"], a["tab"], a["lens"], rows, mb, 12, kv, d,
                                                0.1, a["w"], ws)

    def window(**kw):
        a = dict(good, **kw)
        K.launch_paged_window_attention_decode(a["out"], 12 * d, q, 12 * d, a["pool"], a["tab"], a["lens"], rows, mb, 12, kv, d,
                                               0.1, 9, 0, ws)

    def prefill(**kw):
        a = dict(good, **kw)
        K.launch_paged_window_prefill_attention(a["out"], 12 * d, q, 12 * d, a["pool"], a["tab"], mb, 60, 4, 12, kv, d, 0.1, 9, 0)

    short = dict(w=good["w"][:-1])
    for call in (evict, weights):
        for bad in (short, dict(short, pool=pool.view(-1)), dict(w=good["w"][:1]), dict(w=good["w"].half())):
            with pytest.raises(K.KernelError, match="weights must be"):
                call(**bad)
    for call in (evict, weights, window):
        for bad in (dict(tab=good["tab"].long()), dict(tab=good["tab"][:3]), dict(tab=torch.zeros(rows, 2 * mb, dtype=torch.int32)[:, ::2])):
            with pytest.raises(K.KernelError, match="block_tables must be"):
                call(**bad)
        for bad in (dict(lens=good["lens"].long()), dict(lens=good["lens"][:3])):
            with pytest.raises(K.KernelError, match="seq_lens must be"):
                call(**bad)
    for bad in (dict(dst=good["dst"].long()), dict(dst=good["dst"][:3])):
        with pytest.raises(K.KernelError, match="dst_block_tables must be"):
            evict(**bad)
    for bad in (dict(tab=good["tab"].long()), dict(tab=torch.zeros(3, dtype=torch.int32))):
        with pytest.raises(K.KernelError, match="block_table_row must be"):
            prefill(**bad)
    for call in (weights, window, prefill):
        for bad in (dict(out=good["out"].float()), dict(out=good["out"][:3].clone()), dict(out=torch.zeros(rows, 11 * d, dtype=torch.float16))):
            with pytest.raises(K.KernelError, match="out must hold"):
                call(**bad)
    # rows inside wider ones are fine as long as the last one ends inside the memory
    wide = torch.zeros(rows, 16 * d, dtype=torch.float16)
    K._rows_fit(wide[:, :12 * d], rows, 16 * d, 12 * d)
    K._rows_fit(wide[:, 4 * d:], rows, 16 * d, 12 * d)
    for short in (wide[:, 5 * d:], wide[:1].clone().expand(rows, 16 * d)):
        with pytest.raises(K.KernelError, match="out must hold"):
            K._rows_fit(short, rows, 16 * d, 12 * d)
    for call in (evict, weights):
        with pytest.raises(K.KernelError, match="kv_pool_layer must be contiguous"):
            call(pool=torch.zeros(2 * blocks, 2, kv, 16, d, dtype=torch.float16)[::2])


def test_prompt_launch_plans_are_remembered_for_layers_that_alternate():
    """A launch plan is worked out by replaying the launch, which takes as long as the kernel it is for. Window and full
    attention in turn, or several windows, each find theirs again."""
    def full():
        K.prefill_attention_run_length(6144, 2048, 12, 148)

    def window(w):
        K.window_prefill_workspace_bytes(6144, 2048, 12, w, 4)

    def host_us(calls, n=40):
        best = float("inf")
        for _ in range(5):
            t = time.perf_counter()
            for _ in range(n):
                for f in calls:
                    f()
            best = min(best, time.perf_counter() - t)
        return best / (n * len(calls)) * 1e6

    calls = [full, lambda: window(1024), lambda: window(512), lambda: window(4096)]
    alone = max(host_us([f]) for f in calls)
    assert host_us(calls) < 4 * alone + 4
