"""Bounded-cache operators on the GPU, through the C ABI: attention with a sliding window and sinks (one new token, and
a prompt chunk), decode attention that accumulates each cached token's weight, and eviction by that weight - against
64-bit implementations straight from the definitions.

Tolerances, per output element, from the arithmetic the launchers document (A = sum over visible tokens of p |v|):
  * the output is rounded to FP16 once: half a step, 2^-11 |ref| + 2^-25 for subnormals;
  * probabilities may be rounded to FP16 for P.V: half a step each, 2^-11 A; those below FP16's normal range (against a
    reference at most the row's largest score) lose up to 2^-25 each: 2^-25 sum|v| / sum exp(s - s_max);
  * a score is 128 exact products summed in FP32, off by at most 128 * 2^-24 * scale * sum|q k| (e), its scaling and
    the exponential add a few 2^-24 relative to |s| + 1; numerator and denominator both carry it: 2 (e + ...) A.
For a weight (FP32 sums of probabilities): the same relative terms without the FP16 ones, plus one FP32 rounding of
each addition.
"""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from redline_llm_b200 import kernels as K  # noqa: E402

D, PAGE = 128, 16
SCALE = 1.0 / math.sqrt(D)
INT_MAX = 2**31 - 1
GARBAGE = [0x7E00, 0x7C00, 0xFC00, 0x7C01, 0xFFFF, 0x7BFF]   # NaNs, infinities, the largest finite value


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    K.init()
    yield
    assert K.prefill_attention_health() == 0


def poison(*shape):
    n = math.prod(shape)
    bits = torch.tensor(np.array(GARBAGE, np.uint16).view(np.int16), device="cuda")
    return bits[torch.arange(n, device="cuda") % len(GARBAGE)].view(torch.float16).reshape(shape)


class Cache:
    """One layer's pool with a few sequences in it; everything that is not a live token is poison."""

    def __init__(self, lens, kv_heads, seed, spare=3, extra_pages=0, head_dim=D):
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        self.g, self.lens, self.kv, self.d = g, list(lens), kv_heads, head_dim
        need = [(n + PAGE - 1) // PAGE for n in self.lens]
        self.blocks = sum(need) + 2 + extra_pages
        order = torch.randperm(self.blocks - 2, generator=g, device="cuda") + 2    # 0 padding target, 1 all poison
        self.mbps = max(1, max(need)) + spare
        self.tables = torch.ones(len(self.lens), self.mbps, dtype=torch.int32, device="cuda")
        self.pool = poison(self.blocks, 2, kv_heads, PAGE, head_dim)
        self.slots = []
        at = 0
        for i, n in enumerate(self.lens):
            self.tables[i, :need[i]] = order[at:at + need[i]].int()
            at += need[i]
            t = torch.arange(n, device="cuda")
            block = self.tables[i].long()[t // PAGE]
            self.slots.append((block, t % PAGE))
            self.pool[block, :, :, t % PAGE] = torch.randn(n, 2, kv_heads, head_dim, generator=g, device="cuda").half()
        self.free = order[at:]
        self.seq_lens = torch.tensor(self.lens, dtype=torch.int32, device="cuda")

    def kv64(self, i):
        """[kv_heads, n, d] each, 64 bits."""
        b, s = self.slots[i]
        x = self.pool[b, :, :, s].double()
        return x[:, 0].transpose(0, 1), x[:, 1].transpose(0, 1)

    def hide(self, i, window, sinks):
        """Poisons the tokens of sequence i that a query at its end does not see, and points table entries of pages
        without a visible token at the poison page."""
        n = self.lens[i]
        t = torch.arange(n, device="cuda")
        gone = (t >= sinks) & (t < n - window)
        b, s = self.slots[i]
        self.pool[b[gone], :, :, s[gone]] = poison(int(gone.sum()), 2, self.kv, self.d)
        pages = (n + PAGE - 1) // PAGE
        for page in range(pages):
            if bool(gone[page * PAGE:(page + 1) * PAGE].all()):
                self.tables[i, page] = 1


def attend64(q, k, v, seen, scale=SCALE):
    """q [h, g, d], k / v [h, n, d], seen [n] -> out, tolerance [h, g, d], probabilities [h, g, n] and their tolerance."""
    k, v = k[:, seen], v[:, seen]
    s = torch.einsum("hgd,hnd->hgn", q, k) * scale
    p = torch.softmax(s, dim=2)
    out = torch.einsum("hgn,hnd->hgd", p, v)
    a = torch.einsum("hgn,hnd->hgd", p, v.abs())
    size = torch.einsum("hgd,hnd->hgn", q.abs(), k.abs()).amax(dim=2, keepdim=True) * scale
    rel = 2 * (128 * 2.0**-24 * size + 2.0**-20 * (s.abs().amax(dim=2, keepdim=True) + 1))
    mass = torch.exp(s - s.amax(dim=2, keepdim=True)).sum(dim=2, keepdim=True)
    tol = 2.0**-11 * out.abs() + 2.0**-24 + (2.0**-11 + rel) * a + 2.0**-25 * v.abs().sum(dim=1)[:, None] / mass
    return out, tol, p, p * (rel + 2.0**-23)


def check(got, ref, tol, what):
    assert torch.isfinite(got).all(), f"{what}: something invisible reached a result"
    err = (got.double() - ref).abs()
    assert bool((err <= tol).all()), f"{what}: error {err.max().item():.3e}, {(err / tol).max().item():.2f} of what is allowed"


def decode_case(c, q_heads, window, sinks, seed, q_stride=None, out_stride=None, q_offset=0):
    rows, width = len(c.lens), q_heads * D
    q_stride, out_stride = q_stride or width, out_stride or width
    q = poison(rows + 1, q_stride).clone()
    q[:rows, q_offset:q_offset + width] = torch.randn(rows, width, generator=c.g, device="cuda").half()
    out = torch.full((rows + 1, out_stride), 7.0, dtype=torch.float16, device="cuda")
    return q, out, q_stride, out_stride


def check_decode(c, q, out, q_heads, window, sinks, q_offset=0, what="decode"):
    width = q_heads * D
    for i, n in enumerate(c.lens):
        if n <= 0:
            assert bool((out[i] == 7.0).all()), f"{what}: row {i} without tokens was written"
            continue
        t = torch.arange(n, device="cuda")
        seen = (t < sinks) | (t >= n - window)
        k, v = c.kv64(i)
        ref, tol, _, _ = attend64(q[i, q_offset:q_offset + width].double().view(c.kv, -1, D), k, v, seen)
        check(out[i, :width].view(c.kv, -1, D), ref, tol, f"{what}, sequence {i} of {n}")
        assert bool((out[i, width:] == 7.0).all()), f"{what}: the stride gap was written"
    assert bool((out[len(c.lens):] == 7.0).all()), f"{what}: a row behind the last sequence was written"


LENS = [1, 15, 16, 17, 0, 31, 33, 100, 257, 700, 2051]


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (2, 4), (15, 0), (16, 16), (17, 17), (32, 4), (100, 5), (256, 0),
                                          (257, 300), (511, 33), (2051, 0), (4096, 16), (INT_MAX, INT_MAX), (1, INT_MAX),
                                          (INT_MAX, 0)])
def test_window_decode_over_lengths_windows_and_sinks(window, sinks):
    c = Cache(LENS, 2, seed=window % 1000 + sinks % 7)
    for i in range(len(LENS)):
        c.hide(i, window, sinks)
    q, out, qs, os_ = decode_case(c, 12, window, sinks, 1, q_stride=2048, out_stride=1600, q_offset=128)
    ws = K.window_attention_workspace(len(LENS), c.mbps, 12, 2)
    K.launch_paged_window_attention_decode(out, os_, q, qs, c.pool, c.tables, c.seq_lens, len(LENS), c.mbps, 12, 2, D,
                                           SCALE, window, sinks, ws, q_offset=128)
    check_decode(c, q, out, 12, window, sinks, 128)
    assert K.window_attention_health(ws) == 0


@pytest.mark.parametrize("q_heads,kv_heads", [(1, 1), (2, 1), (3, 3), (8, 1), (10, 2), (7, 1), (28, 4), (64, 8), (8, 8), (15, 3)])
def test_window_decode_head_layouts(q_heads, kv_heads):
    c = Cache([5, 0, 333, 64, 1203], kv_heads, seed=q_heads)
    window, sinks = 200, 3
    for i in range(5):
        c.hide(i, window, sinks)
    q, out, qs, os_ = decode_case(c, q_heads, window, sinks, 2)
    ws = K.window_attention_workspace(5, c.mbps, q_heads, kv_heads)
    K.launch_paged_window_attention_decode(out, os_, q, qs, c.pool, c.tables, c.seq_lens, 5, c.mbps, q_heads, kv_heads, D,
                                           SCALE, window, sinks, ws)
    check_decode(c, q, out, q_heads, window, sinks)


@pytest.mark.parametrize("lens,window", [([32768], 20000), ([20001] * 3 + [40], 16384), (list(range(0, 1300)), 37), ([700], 512),
                                         ([0, 0, 0], 5), ([3] * 65, 2)])
def test_window_decode_batches(lens, window):
    """Long contexts over the whole machine, more sequences than one launch tabulates, batches without any token."""
    c = Cache(lens, 2, seed=len(lens))
    q, out, qs, os_ = decode_case(c, 12, window, 4, 3)
    ws = K.window_attention_workspace(len(lens), c.mbps, 12, 2)
    before = ws.clone() if sum(lens) == 0 else None
    for _ in range(2):
        K.launch_paged_window_attention_decode(out, os_, q, qs, c.pool, c.tables, c.seq_lens, len(lens), c.mbps, 12, 2, D,
                                               SCALE, window, 4, ws)
    check_decode(c, q, out, 12, window, 4)
    if before is not None:
        assert torch.equal(before, ws)
    first = out.clone()
    K.launch_paged_window_attention_decode(out, os_, q, qs, c.pool, c.tables, c.seq_lens, len(lens), c.mbps, 12, 2, D, SCALE,
                                           window, 4, ws)
    assert torch.equal(first, out), "two launches gave different bits"


@pytest.mark.parametrize("lens,q_heads,kv_heads,window,sinks", [
    ([1 + 7 * i % 90 for i in range(41)], 64, 8, 10**6, 0), ([500 + i for i in range(64)], 24, 4, 30, 5),
    ([512 - i % 16 for i in range(80)], 12, 2, 4096, 0),        # 32 pages each: a warp's share of items
    ([513 + i % 3 for i in range(80)], 12, 2, 4096, 0),         # 33
    ([0, 3, 0, 40] * 24, 16, 8, 33, 1), ([20] * 148, 1, 1, 9, 0), ([20] * 149, 1, 1, 9, 0), ([700] * 74, 6, 2, 16, 16)])
def test_decode_many_small_items(lens, q_heads, kv_heads, window, sinks):
    """More (sequence, KV head) items than CTAs, and the shapes around the border of the ways to cut them; window attention
    and weights."""
    c = Cache(lens, kv_heads, seed=len(lens))
    q, out, qs, os_ = decode_case(c, q_heads, 0, 0, 0)
    ws = K.window_attention_workspace(len(lens), c.mbps, q_heads, kv_heads, weights=True)
    for _ in range(2):
        K.launch_paged_window_attention_decode(out, os_, q, qs, c.pool, c.tables, c.seq_lens, len(lens), c.mbps, q_heads, kv_heads, D,
                                               SCALE, window, sinks, ws)
    check_decode(c, q, out, q_heads, window, sinks)
    w = torch.zeros(c.blocks, kv_heads, PAGE, device="cuda")
    out.fill_(7.0)
    K.launch_paged_attention_decode_weights(out, os_, q, qs, c.pool, c.tables, c.seq_lens, len(lens), c.mbps, q_heads, kv_heads, D,
                                            SCALE, w, ws)
    check_decode(c, q, out, q_heads, 10**6, 0)
    ref, tol = weights64(c, q, q_heads, torch.zeros_like(w))
    assert bool(((w.double() - ref).abs() <= tol).all())
    assert K.window_attention_health(ws) == 0


def test_window_decode_lengths_beyond_the_table_are_cut_and_negative_ones_skipped():
    c = Cache([48, 48, 48], 2, seed=5, spare=0)
    c.seq_lens.copy_(torch.tensor([100000, -5, INT_MAX], dtype=torch.int32))
    q, out, qs, os_ = decode_case(c, 12, 20, 2, 4)
    ws = K.window_attention_workspace(3, 3, 12, 2, weights=True)
    K.launch_paged_window_attention_decode(out, os_, q, qs, c.pool, c.tables, c.seq_lens, 3, 3, 12, 2, D, SCALE, 20, 2, ws)
    c.lens = [48, 0, 48]
    check_decode(c, q, out, 12, 20, 2)
    out.fill_(7.0)
    w = torch.zeros(c.blocks, 2, PAGE, device="cuda")
    K.launch_paged_attention_decode_weights(out, os_, q, qs, c.pool, c.tables, c.seq_lens, 3, 3, 12, 2, D, SCALE, w, ws)
    check_decode(c, q, out, 12, 48, 0)
    assert abs(w.sum().item() - 24.0) < 1e-3


def test_a_window_over_everything_agrees_with_the_full_decode_kernel():
    c = Cache([1029, 77, 3000], 2, seed=6)
    q, out, qs, os_ = decode_case(c, 12, 0, 0, 5)
    full = out.clone()
    ws = K.window_attention_workspace(3, c.mbps, 12, 2)
    K.launch_paged_window_attention_decode(out, os_, q, qs, c.pool, c.tables, c.seq_lens, 3, c.mbps, 12, 2, D, SCALE, 3000, 0, ws)
    K.launch_paged_attention_decode(full, os_, q, qs, c.pool, c.tables, c.seq_lens, 3, c.mbps, 12, 2, D, SCALE)
    # two roundings of the same value apart: each is within its own tolerance of the exact one
    assert (out[:3].double() - full[:3].double()).abs().max().item() < 2e-3
    check_decode(c, q, out, 12, 3000, 0)


def test_window_decode_scores_that_outgrow_the_running_maximum():
    """Keys grow by factors of 4 along the context, so the running maximum moves again and again."""
    c = Cache([900], 2, seed=7)
    b, s = c.slots[0]
    for g in range(1, 4):
        c.pool[b[g * 220:], 0, :, s[g * 220:]] *= 4.0
    q, out, qs, os_ = decode_case(c, 12, 0, 0, 6)
    ws = K.window_attention_workspace(1, c.mbps, 12, 2)
    K.launch_paged_window_attention_decode(out, os_, q, qs, c.pool, c.tables, c.seq_lens, 1, c.mbps, 12, 2, D, SCALE, 800, 7, ws)
    check_decode(c, q, out, 12, 800, 7)


def run_prefill(c, q, out, qs, os_, start, rows, q_heads, window, sinks, ws="query", q_offset=0):
    if ws == "query":
        ws = K.window_prefill_workspace(start, rows, q_heads, window, sinks)
    K.launch_paged_window_prefill_attention(out, os_, q, qs, c.pool, c.tables, c.mbps, start, rows, q_heads, c.kv, D, SCALE,
                                            window, sinks, ws, q_offset=q_offset)


def check_prefill(c, q, out, start, rows, q_heads, window, sinks, q_offset=0, some=None):
    width = q_heads * D
    k, v = (x[:, :start + rows] for x in c.kv64(0))
    t = torch.arange(start + rows, device="cuda")
    for i in (range(rows) if some is None else some):
        p = start + i
        seen = (t <= p) & ((t < sinks) | (t > p - window))
        ref, tol, _, _ = attend64(q[i, q_offset:q_offset + width].double().view(c.kv, -1, D), k, v, seen)
        check(out[i, :width].view(c.kv, -1, D), ref, tol, f"row {i} at position {p}")
    assert bool((out[:rows, width:] == 7.0).all()) and bool((out[rows:] == 7.0).all()), "something outside the rows was written"


@pytest.mark.parametrize("start,rows", [(0, 1), (0, 129), (5, 123), (1000, 257), (1024, 128), (2040, 40), (4000, 17)])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 3), (16, 0), (100, 4), (128, 16), (300, 33), (1000, 200), (INT_MAX, 0),
                                          (1, INT_MAX)])
def test_window_prefill_over_chunks_windows_and_sinks(start, rows, window, sinks):
    c = Cache([start + rows], 2, seed=start + rows + sinks % 5)
    # what the chunk's FIRST row no longer sees, no later row sees either
    t = torch.arange(start + rows, device="cuda")
    gone = (t >= sinks) & (t <= start - window)
    b, s = c.slots[0]
    c.pool[b[gone], :, :, s[gone]] = poison(int(gone.sum()), 2, 2, D)
    for page in range((start + rows) // PAGE):
        if bool(gone[page * PAGE:(page + 1) * PAGE].all()):
            c.tables[0, page] = 1
    q, out, qs, os_ = decode_case_rows(c, rows, 12, 2048, 1544, 128)
    run_prefill(c, q, out, qs, os_, start, rows, 12, window, sinks, q_offset=128)
    some = None if rows <= 130 else sorted(set(list(range(0, rows, 7)) + [127, 128, rows - 1]))
    check_prefill(c, q, out, start, rows, 12, window, sinks, 128, some)


def decode_case_rows(c, rows, q_heads, q_stride, out_stride, q_offset=0):
    q = poison(rows + 2, q_stride).clone()
    q[:rows, q_offset:q_offset + q_heads * D] = torch.randn(rows, q_heads * D, generator=c.g, device="cuda").half()
    return q, torch.full((rows + 2, out_stride), 7.0, dtype=torch.float16, device="cuda"), q_stride, out_stride


@pytest.mark.parametrize("q_heads,kv_heads", [(1, 1), (8, 1), (3, 3), (10, 2), (64, 8), (15, 3)])
def test_window_prefill_head_layouts(q_heads, kv_heads):
    c = Cache([700], kv_heads, seed=q_heads + 50)
    q, out, qs, os_ = decode_case_rows(c, 300, q_heads, q_heads * D, q_heads * D)
    run_prefill(c, q, out, qs, os_, 400, 300, q_heads, 150, 5)
    check_prefill(c, q, out, 400, 300, q_heads, 150, 5, some=range(0, 300, 11))


@pytest.mark.parametrize("start,rows,window,sinks", [(9000, 64, 6000, 20), (12000, 130, 12000, 0), (0, 3000, 700, 64)])
def test_window_prefill_cut_across_ctas(start, rows, window, sinks):
    """With a workspace long pairs are cut into runs; without one they are whole: the same function, and each the same
    bits every time."""
    c = Cache([start + rows], 2, seed=rows)
    q, out, qs, os_ = decode_case_rows(c, rows, 12, 1536, 1536)
    whole, again = out.clone(), out.clone()
    assert rows == 3000 or K.window_prefill_workspace_bytes(start, rows, 12, window, sinks) > 0
    run_prefill(c, q, out, qs, os_, start, rows, 12, window, sinks)
    run_prefill(c, q, again, qs, os_, start, rows, 12, window, sinks)
    run_prefill(c, q, whole, qs, os_, start, rows, 12, window, sinks, ws=None)
    assert torch.equal(out, again)
    some = sorted({0, 1, rows // 2, rows - 2, rows - 1})
    check_prefill(c, q, out, start, rows, 12, window, sinks, some=some)
    check_prefill(c, q, whole, start, rows, 12, window, sinks, some=some)


def test_window_prefill_scores_that_outgrow_the_reference():
    c = Cache([1400], 2, seed=77)
    b, s = c.slots[0]
    for at, f in ((640, 8.0), (900, 4.0), (1100, 4.0)):
        c.pool[b[at:], 0, :, s[at:]] *= f
    q, out, qs, os_ = decode_case_rows(c, 400, 12, 1536, 1536)
    run_prefill(c, q, out, qs, os_, 1000, 400, 12, 600, 40)
    check_prefill(c, q, out, 1000, 400, 12, 600, 40, some=range(0, 400, 13))


@pytest.mark.parametrize("window,sinks", [(20, 1), (1, 1), (40, 0), (5000, 0)])
def test_a_visible_key_of_minus_infinity_has_weight_zero(window, sinks):
    """The first and the newest token score -inf; each may be all that its page shows."""
    lens = [17, 33, 300, 16, 2001, 4993]
    c = Cache(lens, 2, seed=sinks + 3)
    for i, n in enumerate(lens):
        b, s = c.slots[i]
        for t in (0, n - 1):
            if (window, sinks) != (1, 1) or t > 0:   # one visible key has to be finite
                c.pool[b[t], 0, :, s[t], 0] = float("-inf")
    q, out, qs, os_ = decode_case(c, 12, 0, 0, 0)
    q[:len(lens)].view(len(lens), 12, D)[:, :, 0] = 0.5
    ws = K.window_attention_workspace(len(lens), c.mbps, 12, 2, weights=True)
    w = torch.zeros(c.blocks, 2, PAGE, device="cuda")

    def verify(window, sinks, weights):
        for i, n in enumerate(lens):
            t = torch.arange(n, device="cuda")
            k, v = c.kv64(i)
            seen = ((t < sinks) | (t >= n - window)) & torch.isfinite(k[0, :, 0])
            ref, tol, p, ptol = attend64(q[i, :12 * D].double().view(2, -1, D), k, v, seen)
            check(out[i].view(2, -1, D), ref, tol, f"sequence {i} of {n}")
            if weights:
                b, s = c.slots[i]
                got = w[b, :, s].T.double()
                want, room = torch.zeros_like(got), torch.zeros_like(got)
                want[:, seen], room[:, seen] = p.sum(1), ptol.sum(1) + 9 * 2.0**-24 * p.sum(1)
                assert bool(((got - want).abs() <= room).all())

    K.launch_paged_attention_decode_weights(out, os_, q, qs, c.pool, c.tables, c.seq_lens, len(lens), c.mbps, 12, 2, D, SCALE, w, ws)
    verify(5000, 0, True)
    K.launch_paged_window_attention_decode(out, os_, q, qs, c.pool, c.tables, c.seq_lens, len(lens), c.mbps, 12, 2, D, SCALE, window,
                                           sinks, ws)
    verify(window, sinks, False)


@pytest.mark.parametrize("start,rows,window,sinks", [(1000, 200, 100, 1), (0, 300, 50, 2), (6000, 64, 5000, 1)])
def test_window_prefill_visible_keys_of_minus_infinity(start, rows, window, sinks):
    """The sinks score -inf: for later rows of a tile they are all that the first block of keys shows."""
    c = Cache([start + rows], 2, seed=rows)
    b, s = c.slots[0]
    first = sinks if start else sinks - 1   # from position 0 on, the first row sees nothing else
    c.pool[b[sinks - first:sinks], 0, :, s[sinks - first:sinks], 0] = float("-inf")
    q, out, qs, os_ = decode_case_rows(c, rows, 12, 1536, 1536)
    q[:rows].view(rows, 12, D)[:, :, 0] = 0.5
    run_prefill(c, q, out, qs, os_, start, rows, 12, window, sinks)
    k, v = c.kv64(0)
    t = torch.arange(start + rows, device="cuda")
    for i in range(0, rows, 9):
        p = start + i
        seen = (t <= p) & ((t < sinks) | (t > p - window)) & torch.isfinite(k[0, :, 0])
        ref, tol, _, _ = attend64(q[i, :12 * D].double().view(2, -1, D), k, v, seen)
        check(out[i].view(2, -1, D), ref, tol, f"row {i}")


def weights64(c, q, q_heads, old):
    """Expected weights and their tolerance after one step, from the old ones."""
    new, tol = old.double().clone(), torch.zeros_like(old, dtype=torch.float64)
    for i, n in enumerate(c.lens):
        if n <= 0:
            continue
        k, v = c.kv64(i)
        _, _, p, ptol = attend64(q[i, :q_heads * D].double().view(c.kv, -1, D), k, v, torch.ones(n, dtype=torch.bool, device="cuda"))
        b, s = c.slots[i]
        prev = old.double()[b, :, s]
        prev[n - 1] = 0.0
        now = prev + p.sum(dim=1).T
        new[b, :, s] = now
        tol[b, :, s] = ptol.sum(dim=1).T + 9 * 2.0**-24 * now.abs()
    return new, tol


@pytest.mark.parametrize("lens,q_heads,kv_heads", [([1], 12, 2), ([16, 0, 17, 300], 12, 2), ([1031], 5, 1), ([2, 900, 33], 64, 8),
                                                   ([40, 41], 9, 3), ([20000, 12], 12, 2), (list(range(0, 1100)), 2, 1)])
def test_weights_decode(lens, q_heads, kv_heads):
    c = Cache(lens, kv_heads, seed=len(lens) + q_heads)
    q, out, qs, os_ = decode_case(c, q_heads, 0, 0, 8)
    w = torch.full((c.blocks, kv_heads, PAGE), float("nan"), device="cuda")
    for i, n in enumerate(lens):
        b, s = c.slots[i]
        w[b[:-1], :, s[:-1]] = torch.rand(max(0, n - 1), kv_heads, generator=c.g, device="cuda")   # the newest stays NaN
    old = w.clone()
    ws = K.window_attention_workspace(len(lens), c.mbps, q_heads, kv_heads, weights=True)
    K.launch_paged_attention_decode_weights(out, os_, q, qs, c.pool, c.tables, c.seq_lens, len(lens), c.mbps, q_heads,
                                            kv_heads, D, SCALE, w, ws)
    check_decode(c, q, out, q_heads, INT_MAX, 0, what="weights decode")
    ref, tol = weights64(c, q, q_heads, old)
    live = torch.zeros_like(w, dtype=torch.bool)
    for b, s in c.slots:
        live[b, :, s] = True
    assert bool(((w.double() - ref).abs() <= tol)[live].all())
    assert bool(torch.isnan(w[~live]).all()), "an entry of no cached token was written"
    twice = old.clone()
    K.launch_paged_attention_decode_weights(out, os_, q, qs, c.pool, c.tables, c.seq_lens, len(lens), c.mbps, q_heads,
                                            kv_heads, D, SCALE, twice, ws)
    assert torch.equal(torch.nan_to_num(w, nan=-1.0), torch.nan_to_num(twice, nan=-1.0)), "two launches gave different bits"
    assert K.window_attention_health(ws) == 0


def evict64(w, table, n, budget, sinks, recent):
    """Kept slots of one sequence and head, by a stable sort of the definition's order."""
    m = min(n, budget)
    if n <= budget:
        return np.arange(m)
    rest = np.arange(sinks, n - recent)
    x = w[rest].astype(np.float64)
    x = np.where(np.isnan(x), -np.inf, x)
    low = np.isnan(w[rest])                         # below even -inf
    order = np.lexsort((rest, -x, low))             # numbers before NaN, heavier first, then the lower position
    keep = rest[np.array(order[:m - sinks - recent], dtype=np.int64)]
    return np.sort(np.concatenate([np.arange(sinks), keep, np.arange(n - recent, n)]).astype(np.int64))


def check_evict(c, budget, sinks, recent, w, in_place, alias=False, spare_dst=0):
    kv, rows = c.kv, len(c.lens)
    pool0, w0 = c.pool.clone(), w.clone()
    if in_place:
        dst, dmb = c.tables, c.mbps
    else:
        per = (budget + PAGE - 1) // PAGE
        dmb = per + spare_dst
        dst = torch.zeros(rows, dmb, dtype=torch.int32, device="cuda")
        assert len(c.free) >= rows * per
        dst[:, :per] = c.free[:rows * per].view(rows, per).int()
    kept = torch.full((rows, kv, budget), -9, dtype=torch.int32, device="cuda")
    new = c.seq_lens if alias else torch.full((rows + 1,), -9, dtype=torch.int32, device="cuda")
    K.launch_kv_evict(c.pool, w, c.tables, c.mbps, dst, dmb, c.seq_lens, new, kept, rows, kv, c.d, budget, sinks, recent)
    torch.cuda.synchronize()
    want_pool, want_w = pool0.view(torch.int16).clone(), w0.view(torch.int32).clone()
    for i, n in enumerate(c.lens):
        n = max(0, n)
        m = min(n, budget)
        assert int(new[i]) == m
        b, s = c.slots[i]
        to_b, to_s = dst[i].long()[torch.arange(m, device="cuda") // PAGE], torch.arange(m, device="cuda") % PAGE
        for h in range(kv):
            keep = evict64(w0[b, h, s].cpu().numpy(), None, n, budget, sinks, recent)
            assert np.array_equal(kept[i, h, :m].cpu().numpy(), keep), f"sequence {i} head {h}"
            assert bool((kept[i, h, m:] == -1).all())
            keep = torch.from_numpy(keep).cuda()
            want_pool[to_b, :, h, to_s] = pool0.view(torch.int16)[b[keep], :, h, s[keep]]
            want_w[to_b, h, to_s] = w0.view(torch.int32)[b[keep], h, s[keep]]
    assert torch.equal(c.pool.view(torch.int16), want_pool), "pool"
    assert torch.equal(w.view(torch.int32), want_w), "weights"
    if not alias:
        assert int(new[rows]) == -9
    return kept


def some_weights(c, kind):
    u = torch.rand(c.blocks, c.kv, PAGE, generator=c.g, device="cuda")
    if kind == "ties":
        return (u * 4).floor()
    if kind == "equal":
        return torch.full_like(u, 0.25)
    if kind == "crowded":                    # nearly all in one part in two thousand of the range, many of them equal
        w = 1.0 + (u * 500).floor() * 1e-6
        w[u < 0.002] = 1e30
        w[(u > 0.5) & (u < 0.501)] = -1e30
        return w
    if kind == "odd":
        w = u - 0.5
        w[u < 0.2] = float("nan")
        w[(u > 0.2) & (u < 0.3)] = float("inf")
        w[(u > 0.3) & (u < 0.4)] = float("-inf")
        w[(u > 0.4) & (u < 0.5)] = 0.0
        w[(u > 0.5) & (u < 0.6)] = -0.0
        w[(u > 0.6) & (u < 0.7)] *= 1e-38
        return w
    return u.pow(-0.7) - 0.99


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("kind", ["spread", "ties", "equal", "odd"])
@pytest.mark.parametrize("budget,sinks,recent", [(1, 0, 0), (1, 1, 0), (1, 0, 1), (16, 4, 4), (17, 0, 17), (100, 4, 30), (256, 0, 0),
                                                 (255, 255, 0), (300, 17, 33)])
def test_evict(budget, sinks, recent, kind, in_place):
    lens = [1, 16, 0, 17, 100, 255, 256, 257, 1030, 301]
    c = Cache(lens, 2, seed=budget + sinks, extra_pages=len(lens) * 20, spare=max(1, 20))
    check_evict(c, budget, sinks, recent, some_weights(c, kind), in_place, alias=kind == "ties")


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("lens,kv,budget,sinks,recent", [([32768], 2, 8191, 4, 100), ([5000, 70000], 1, 4100, 0, 0), ([3000] * 9, 8, 2999, 0, 10),
                                                         ([700] * 70, 4, 64, 4, 20)])
def test_evict_sizes(lens, kv, budget, sinks, recent, in_place):
    c = Cache(lens, kv, seed=kv, extra_pages=len(lens) * ((budget + 15) // 16), head_dim=D)
    check_evict(c, budget, sinks, recent, some_weights(c, "spread"), in_place)


@pytest.mark.parametrize("lens,kv,budget", [([6000, 3000], 1, 1500), ([9000] * 40, 2, 4000), ([30000], 2, 9000)])
def test_evict_weights_that_share_a_bin(lens, kv, budget):
    """Thousands of candidates fall into one bin of the first division, with and without a cluster per item."""
    c = Cache(lens, kv, seed=kv + 7)
    check_evict(c, budget, 4, 100, some_weights(c, "crowded"), True)


@pytest.mark.parametrize("rows,kv", [(96, 8), (10, 2)])
def test_evict_rank_after_a_second_division(rows, kv):
    """The limit lies among 500 neighbours that share a bin of the first division and are divided once more before the
    last few are ranked: every warp must have read the count of its bin by then. Many items at once, again and again."""
    n, budget = 2000, 1000
    c = Cache([n] * rows, kv, seed=rows, spare=1)
    band = 1.0 + torch.arange(500, device="cuda").double() * 2.0**-16   # apart by far more than an fp32 step
    rest = torch.cat([torch.linspace(-1e4, -1e3, 750), torch.linspace(1e3, 1e4, 750)]).cuda().double()
    values = torch.cat([band, rest]).float()
    w = torch.zeros(c.blocks, kv, PAGE, device="cuda")
    keep = torch.empty(rows, kv, budget, dtype=torch.int32, device="cuda")
    for i, (b, s) in enumerate(c.slots):
        for h in range(kv):
            x = values[torch.randperm(n, generator=c.g, device="cuda")]
            w[b, h, s] = x
            keep[i, h] = torch.nonzero(x > x.sort().values[n - budget - 1]).flatten().int()
    kept = torch.empty_like(keep)
    new = torch.empty(rows, dtype=torch.int32, device="cuda")
    for _ in range(20):
        weights = w.clone()   # the selection reads these; what the pool holds does not matter here
        kept.fill_(-9)
        K.launch_kv_evict(c.pool, weights, c.tables, c.mbps, c.tables, c.mbps, c.seq_lens, new, kept, rows, kv, c.d, budget, 0, 0)
        assert torch.equal(kept, keep)


@pytest.mark.parametrize("rows,kv,budget,head_dim", [(n, kv, budget, d) for d in (D, 64) for n, kv in ((3, 2), (9, 4), (70, 2))
                                                     for budget in (1, 8, 17, 64, 65, 130, 257, 513, 1025)])
def test_evict_in_place_around_a_round(rows, kv, budget, head_dim):
    """In place, clusters of one to eight CTAs: kept tokens at and next to what a CTA or a cluster has in registers."""
    c = Cache([1100 + i % 7 for i in range(rows)], kv, seed=budget, head_dim=head_dim)
    check_evict(c, budget, 0, 1, some_weights(c, "spread"), True, alias=True)


def test_evict_more_tokens_than_shared_memory_holds():
    """80 items, so one CTA each, two of them longer than the keys that a CTA keeps."""
    c = Cache([47001, 50] + [100] * 8, 8, seed=12)
    check_evict(c, 700, 4, 20, some_weights(c, "spread"), True)
    c = Cache([47001, 50] + [100] * 8, 8, seed=13)
    check_evict(c, 40000, 0, 0, some_weights(c, "ties"), True)


@pytest.mark.parametrize("spare", [0, 1400, 1500, 2600])
def test_evict_more_items_than_sms_in_tables_of_any_width(spare):
    """160 items in tables whose width lets two selections share an SM or not, and behind what shared memory holds."""
    c = Cache([40 + 13 * i for i in range(20)], 8, seed=spare, spare=spare)
    check_evict(c, 150, 4, 30, some_weights(c, "spread"), True)


@pytest.mark.parametrize("head_dim", [8, 64, 96, 256, 1024])
def test_evict_row_widths(head_dim):
    c = Cache([90, 200], 3, seed=head_dim, extra_pages=40, head_dim=head_dim)
    check_evict(c, 77, 3, 20, some_weights(c, "spread"), False, spare_dst=3)
    c = Cache([90, 200], 3, seed=head_dim, head_dim=head_dim)
    check_evict(c, 77, 3, 20, some_weights(c, "spread"), True)


def test_offsets_past_32_bits():
    """A pool slice of more than 2^32 bytes with every page of the sequence at its far end."""
    pages, blocks, kv = 40, 140000, 8
    pool = torch.empty(blocks, 2, kv, PAGE, D, dtype=torch.float16, device="cuda")     # 9.2 GB, 4.6e9 elements
    n = pages * PAGE - 3
    c = Cache([n], kv, seed=9, spare=0)
    far = torch.arange(blocks - c.blocks, blocks, device="cuda")
    pool[far] = c.pool
    c.pool, c.tables = pool, c.tables + (blocks - c.blocks)
    c.slots = [(c.slots[0][0] + (blocks - c.blocks), c.slots[0][1])]
    w = torch.zeros(blocks, kv, PAGE, device="cuda")
    q, out, qs, os_ = decode_case(c, 64, 0, 0, 10)
    ws = K.window_attention_workspace(1, c.mbps, 64, kv, weights=True)
    K.launch_paged_window_attention_decode(out, os_, q, qs, pool, c.tables, c.seq_lens, 1, c.mbps, 64, kv, D, SCALE, 300, 20, ws)
    check_decode(c, q, out, 64, 300, 20)
    K.launch_paged_attention_decode_weights(out, os_, q, qs, pool, c.tables, c.seq_lens, 1, c.mbps, 64, kv, D, SCALE, w, ws)
    check_decode(c, q, out, 64, n, 0)
    assert abs(w.double().sum().item() - 64.0) < 1e-3
    q, out, qs, os_ = decode_case_rows(c, 60, 64, 64 * D, 64 * D)
    run_prefill(c, q, out, qs, os_, n - 60, 60, 64, 200, 9)
    check_prefill(c, q, out, n - 60, 60, 64, 200, 9, some=[0, 31, 59])
    want = pool[c.slots[0][0], :, :, c.slots[0][1]].clone()
    kept = torch.zeros(1, kv, 100, dtype=torch.int32, device="cuda")
    K.launch_kv_evict(pool, w, c.tables, c.mbps, c.tables, c.mbps, c.seq_lens, c.seq_lens, kept, 1, kv, D, 100, 4, 30)
    b, s = c.slots[0][0][:100], c.slots[0][1][:100]
    for h in range(kv):
        assert torch.equal(pool[b, :, h, s], want[kept[0, h].long(), :, h])


def test_one_workspace_serves_different_calls_in_order_and_graphs_replay_them():
    shapes = [([700], 512), ([5, 900, 0, 33], 100), (list(range(1, 60)), 20)]
    ws = K.window_attention_workspace(59, 200, 12, 2, weights=True)
    cases = [Cache(l, 2, seed=40 + i) for i, (l, _) in enumerate(shapes)]
    io = [decode_case(c, 12, 0, 0, 0) for c in cases]
    w = [torch.zeros(c.blocks, 2, PAGE, device="cuda") for c in cases]

    def go():
        for c, (q, out, qs, os_), (l, window), wt in zip(cases, io, shapes, w):
            K.launch_paged_attention_decode_weights(out, os_, q, qs, c.pool, c.tables, c.seq_lens, len(l), c.mbps, 12, 2, D,
                                                    SCALE, wt, ws)
            K.launch_paged_window_attention_decode(out, os_, q, qs, c.pool, c.tables, c.seq_lens, len(l), c.mbps, 12, 2, D,
                                                   SCALE, window, 4, ws)

    go()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        go()
    for x in w:
        x.zero_()
    for c, (q, out, _, _), (l, _) in zip(cases, io, shapes):
        out.fill_(7.0)
        q[:len(l), :1536] = torch.randn(len(l), 1536, generator=c.g, device="cuda").half()     # new inputs, same buffers
    for _ in range(3):
        g.replay()
    torch.cuda.synchronize()
    for c, (q, out, _, _), (l, window), wt in zip(cases, io, shapes, w):
        check_decode(c, q, out, 12, window, 4)
        one, tol = weights64(c, q, 12, torch.zeros_like(wt))
        for i, n in enumerate(l):
            if n == 0:
                continue
            b, s = c.slots[i]
            times = torch.full((n, 1), 3.0, device="cuda", dtype=torch.float64)
            times[n - 1] = 1.0                                                                  # the newest starts over
            assert bool(((wt.double() - 0)[b, :, s] - times * one[b, :, s]).abs().le(3 * tol[b, :, s] + 1e-6 * one[b, :, s]).all())
    assert K.window_attention_health(ws) == 0


def test_streams_with_a_workspace_each():
    cases = [Cache([3000, 1200], 2, seed=60), Cache([2500, 40, 900], 2, seed=61)]
    io = [decode_case(c, 12, 0, 0, 0) for c in cases]
    ws = [K.window_attention_workspace(len(c.lens), c.mbps, 12, 2) for c in cases]
    pf = [decode_case_rows(Cache([10], 2, seed=62), 200, 12, 1536, 1536) for _ in cases]
    pws = [K.window_prefill_workspace(700, 200, 12, 600, 4) for _ in cases]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(10):
        for c, (q, out, qs, os_), x, (pq, pout, pqs, pos_), px, st in zip(cases, io, ws, pf, pws, streams):
            K.launch_paged_window_attention_decode(out, os_, q, qs, c.pool, c.tables, c.seq_lens, len(c.lens), c.mbps, 12, 2,
                                                   D, SCALE, 1000, 4, x, stream=st)
            K.launch_paged_window_prefill_attention(pout, pos_, pq, pqs, c.pool, c.tables, c.mbps, 700, 200, 12, 2, D, SCALE,
                                                    600, 4, px, stream=st)
    torch.cuda.synchronize()
    for c, (q, out, _, _), (pq, pout, _, _) in zip(cases, io, pf):
        check_decode(c, q, out, 12, 1000, 4)
        check_prefill(c, pq, pout, 700, 200, 12, 600, 4, some=[0, 100, 199])


@pytest.mark.parametrize("shift,stride", [(0, 1537), (1, 1538), (2, 1540), (4, 1540)])
def test_decode_output_rows_of_any_alignment(shift, stride):
    c = Cache([700, 90], 2, seed=70)
    q, _, qs, _ = decode_case(c, 12, 0, 0, 0)
    buf = torch.full((3 * stride + 8,), 7.0, dtype=torch.float16, device="cuda")
    out = buf[shift:shift + 3 * stride].view(3, stride)
    ws = K.window_attention_workspace(2, c.mbps, 12, 2)
    K.launch_paged_window_attention_decode(out, stride, q, qs, c.pool, c.tables, c.seq_lens, 2, c.mbps, 12, 2, D, SCALE, 300, 4, ws)
    check_decode(c, q, out, 12, 300, 4)
    assert bool((buf[:shift] == 7.0).all()) and bool((buf[shift + 3 * stride:] == 7.0).all())


@pytest.mark.parametrize("lens", [[700, 33, 1500], [900 + i for i in range(70)] + [8000] * 3, [5 + i for i in range(90)]],
                         ids=["chunks", "shares", "teams"])
def test_a_wait_that_runs_out_is_reported_and_the_next_launch_is_right(lens):
    """The give-up path of the decode kernels' bounded waits, for each way to deal the pages: through the test hook one
    warp never requests its first page, so its wait (shortened to about a millisecond) runs out. The launch comes back,
    rl_window_attention_health says so once, and the next ordinary launch on the same workspace is correct."""
    c = Cache(lens, 2, seed=len(lens))
    rows = len(lens)
    q, out, qs, os_ = decode_case(c, 12, 0, 0, 0)
    ws = K.window_attention_workspace(rows, c.mbps, 12, 2, weights=True)
    w = torch.zeros(c.blocks, 2, PAGE, device="cuda")

    def window():
        K.launch_paged_window_attention_decode(out, os_, q, qs, c.pool, c.tables, c.seq_lens, rows, c.mbps, 12, 2, D, SCALE, 10**6, 0, ws)

    def weights():
        K.launch_paged_attention_decode_weights(out, os_, q, qs, c.pool, c.tables, c.seq_lens, rows, c.mbps, 12, 2, D, SCALE, w, ws)

    for launch in (window, weights):
        try:
            K.attention_test_wait_expiry(True, 2_000_000)
            launch()
            assert K.window_attention_health(ws) == 1, "the wait that ran out was not reported"
            assert K.window_attention_health(ws) == 0, "the flag is cleared by the query that reported it"
        finally:
            K.attention_test_wait_expiry(False, 0)
        out.fill_(7.0)
        launch()
        check_decode(c, q, out, 12, 10**6, 0)
        assert K.window_attention_health(ws) == 0


def test_tensors_elsewhere_are_refused():
    c = Cache([40], 2, seed=71)
    q, out, qs, os_ = decode_case(c, 12, 0, 0, 0)
    ws = K.window_attention_workspace(1, c.mbps, 12, 2, weights=True)
    w = torch.zeros(c.blocks, 2, PAGE, device="cuda")
    kept = torch.zeros(1, 2, 16, dtype=torch.int32, device="cuda")
    with pytest.raises(K.KernelError):
        K.launch_paged_window_attention_decode(out, os_, q.cpu(), qs, c.pool, c.tables, c.seq_lens, 1, c.mbps, 12, 2, D, SCALE, 9, 0, ws)
    with pytest.raises(K.KernelError):
        K.launch_paged_attention_decode_weights(out, os_, q, qs, c.pool, c.tables, c.seq_lens.cpu(), 1, c.mbps, 12, 2, D, SCALE, w, ws)
    with pytest.raises(K.KernelError):
        K.launch_paged_window_prefill_attention(out, os_, q, qs, c.pool, c.tables.cpu(), c.mbps, 39, 1, 12, 2, D, SCALE, 9, 0, None)
    with pytest.raises(K.KernelError):
        K.launch_kv_evict(c.pool, w.cpu(), c.tables, c.mbps, c.tables, c.mbps, c.seq_lens, c.seq_lens, kept, 1, 2, D, 16, 0, 0)
    assert bool((out == 7.0).all())


def test_prompt_attention_and_eviction_in_graphs():
    """Captured and replayed: a chunk cut into runs, and an eviction to other pages; the same bits as when launched."""
    c = Cache([9000], 2, seed=72, extra_pages=80)
    pq, pout, pqs, pos_ = decode_case_rows(c, 64, 12, 1536, 1536)
    pws = K.window_prefill_workspace(8936, 64, 12, 6000, 20)
    assert K.window_prefill_workspace_bytes(8936, 64, 12, 6000, 20) > 0, "this chunk is meant to be cut"
    w = some_weights(c, "spread")
    dst = c.free[:63].view(1, 63).int().contiguous()
    new = torch.zeros(1, dtype=torch.int32, device="cuda")
    kept = torch.zeros(1, 2, 1000, dtype=torch.int32, device="cuda")

    def go():
        run_prefill(c, pq, pout, pqs, pos_, 8936, 64, 12, 6000, 20, ws=pws)
        K.launch_kv_evict(c.pool, w, c.tables, c.mbps, dst, 63, c.seq_lens, new, kept, 1, 2, D, 1000, 4, 100)

    go()
    want = [x.clone() for x in (pout, c.pool.view(torch.int16), w.view(torch.int32), new, kept)]
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        go()
    pout.fill_(7.0)
    new.zero_()
    kept.zero_()
    c.pool[dst[0].long()] = 0
    for _ in range(3):
        g.replay()
    torch.cuda.synchronize()
    assert bool((pout[:64] == want[0][:64]).all()) and torch.equal(new, want[3]) and torch.equal(kept, want[4])
    live = torch.arange(1000, device="cuda")
    b, sl = dst[0].long()[live // PAGE], live % PAGE
    assert torch.equal(c.pool.view(torch.int16)[b, :, :, sl], want[1][b, :, :, sl])
    assert torch.equal(w.view(torch.int32), want[2])


def test_with_dependent_launch_on_a_step_sees_what_the_launches_before_it_wrote():
    """rl_attention_set_prologue_overlap: scatter, weights, window attention and an eviction in place back to back, launched
    many times without a pause, and in a graph - the same bits as with the option off."""
    def loop(overlap, graph):
        K.set_attention_prologue_overlap(overlap)
        try:
            c = Cache([900, 1500, 64], 2, seed=80)
            g = torch.Generator(device="cuda")
            g.manual_seed(81)
            rows, heads, kv = 3, 12, 2
            fresh = [torch.randn(rows, kv * D, generator=g, device="cuda").half() for _ in range(12)]
            q = torch.randn(rows, heads * D, generator=g, device="cuda").half()
            w = torch.rand(c.blocks, kv, PAGE, generator=g, device="cuda")
            outs = [torch.zeros(rows, heads * D, dtype=torch.float16, device="cuda") for _ in range(18)]
            kept = torch.zeros(rows, kv, 800, dtype=torch.int32, device="cuda")
            ws = K.window_attention_workspace(rows, c.mbps, heads, kv, weights=True)
            lens0, pool0, w0 = c.seq_lens.clone(), c.pool.clone(), w.clone()
            pos = c.seq_lens - 1

            def go():
                for i in range(6):
                    K.launch_kv_scatter(c.pool, fresh[2 * i], fresh[2 * i + 1], kv * D, kv * D, c.tables, c.mbps, pos, rows, kv, D)
                    K.launch_paged_attention_decode_weights(outs[3 * i], heads * D, q, heads * D, c.pool, c.tables, c.seq_lens, rows,
                                                            c.mbps, heads, kv, D, SCALE, w, ws)
                    K.launch_paged_window_attention_decode(outs[3 * i + 1], heads * D, q, heads * D, c.pool, c.tables, c.seq_lens,
                                                           rows, c.mbps, heads, kv, D, SCALE, 200, 4, ws)
                    if i == 2:
                        K.launch_kv_evict(c.pool, w, c.tables, c.mbps, c.tables, c.mbps, c.seq_lens, c.seq_lens, kept, rows, kv, D,
                                          800, 4, 100)
                    K.launch_paged_window_attention_decode(outs[3 * i + 2], heads * D, q, heads * D, c.pool, c.tables, c.seq_lens,
                                                           rows, c.mbps, heads, kv, D, SCALE, 10000, 0, ws)
                    pos.copy_(c.seq_lens - 1)

            torch.cuda.synchronize()
            if graph:
                go()
                torch.cuda.synchronize()
                cg = torch.cuda.CUDAGraph()
                with torch.cuda.graph(cg):
                    go()
                run = cg.replay
            else:
                run = go
            for _ in range(5):
                c.seq_lens.copy_(lens0)
                c.pool.view(torch.int16).copy_(pool0.view(torch.int16))
                w.copy_(w0)
                pos.copy_(lens0 - 1)
                torch.cuda.synchronize()
                run()
                torch.cuda.synchronize()
                yield [x.clone() for x in outs] + [c.pool.view(torch.int16).clone(), w.view(torch.int32).clone(), c.seq_lens.clone(), kept.clone()]
        finally:
            K.set_attention_prologue_overlap(False)

    want = next(iter(loop(False, False)))
    for overlap, graph in ((False, True), (True, False), (True, True)):
        for got in loop(overlap, graph):
            for a, b in zip(want, got):
                assert torch.equal(a.nan_to_num(7.0) if a.is_floating_point() else a, b.nan_to_num(7.0) if b.is_floating_point() else b)


@pytest.mark.parametrize("in_place", [True, False])
def test_the_overlap_option_may_change_between_an_eviction_and_the_decode_behind_it(in_place):
    """Launched with the option off, and the decode behind it with the option on: it reads lengths and older pages ahead of
    its wait, and has to see the moved ones."""
    rows, kv, heads, budget = 40, 2, 12, 1024
    outs = []
    for overlap in (False, True):
        got = []
        for run in range(8):
            c = Cache([3000 + 7 * i for i in range(rows)], kv, seed=90, extra_pages=rows * budget // PAGE)
            w = some_weights(c, "spread")
            dst = c.tables if in_place else c.free[:rows * budget // PAGE].view(rows, -1).int().contiguous()
            mb = dst.shape[1]
            q, out, qs, os_ = decode_case(c, heads, 0, 0, 0)
            kept = torch.zeros(rows, kv, budget, dtype=torch.int32, device="cuda")
            ws = K.window_attention_workspace(rows, c.mbps, heads, kv)
            torch.cuda.synchronize()
            K.launch_kv_evict(c.pool, w, c.tables, c.mbps, dst, mb, c.seq_lens, c.seq_lens, kept, rows, kv, D, budget, 4, 100)
            K.set_attention_prologue_overlap(overlap)
            try:
                K.launch_paged_window_attention_decode(out, os_, q, qs, c.pool, dst, c.seq_lens, rows, mb, heads, kv, D, SCALE, 10**6, 0, ws)
            finally:
                K.set_attention_prologue_overlap(False)
            got.append(out.clone())
        outs.append(got)
    for x in outs[0] + outs[1]:
        assert torch.equal(x, outs[0][0])


@pytest.mark.parametrize("in_place", [True, False])
def test_both_decode_kernels_read_moved_pages_early(in_place):
    """With the overlap option on, decode launches right behind an eviction request the moved rows by tensor copies ahead of
    their wait: the same bits as with the option off, for the full and the window kernel, through graph replays."""
    rows, kv, heads, budget = 24, 2, 12, 512
    c = Cache([1200 + 31 * i for i in range(rows)], kv, seed=91, extra_pages=rows * budget // PAGE)
    w = some_weights(c, "spread")
    dst = c.tables if in_place else c.free[:rows * budget // PAGE].view(rows, -1).int().contiguous()
    mb = dst.shape[1]
    q, full, qs, os_ = decode_case(c, heads, 0, 0, 0)
    window = full.clone()
    new = torch.zeros_like(c.seq_lens)
    kept = torch.zeros(rows, kv, budget, dtype=torch.int32, device="cuda")
    ws = K.window_attention_workspace(rows, c.mbps, heads, kv)
    lens0, pool0, w0 = c.seq_lens.clone(), c.pool.clone(), w.clone()

    def go(first, second):
        K.launch_kv_evict(c.pool, w, c.tables, c.mbps, dst, mb, c.seq_lens, new, kept, rows, kv, D, budget, 4, 100)
        for name in (first, second):
            if name == "full":
                K.launch_paged_attention_decode(full, os_, q, qs, c.pool, dst, new, rows, mb, heads, kv, D, SCALE)
            else:
                K.launch_paged_window_attention_decode(window, os_, q, qs, c.pool, dst, new, rows, mb, heads, kv, D, SCALE, 300, 4, ws)

    results = []
    for overlap in (False, True):
        K.set_attention_prologue_overlap(overlap)
        try:
            for order in (("full", "window"), ("window", "full")):
                g = torch.cuda.CUDAGraph()
                go(*order)
                torch.cuda.synchronize()
                with torch.cuda.graph(g):
                    go(*order)
                for _ in range(6):
                    c.pool.view(torch.int16).copy_(pool0.view(torch.int16))
                    w.copy_(w0)
                    new.zero_()
                    full.fill_(7.0), window.fill_(7.0)
                    torch.cuda.synchronize()
                    g.replay()
                    torch.cuda.synchronize()
                    results.append((full.clone(), window.clone()))
        finally:
            K.set_attention_prologue_overlap(False)
    assert torch.equal(c.seq_lens, lens0)
    for a, b in results:
        assert torch.isfinite(a[:rows]).all() and torch.equal(a, results[0][0]) and torch.equal(b, results[0][1])


@pytest.mark.parametrize("kernel", ["full", "window", "weights"])
def test_a_decode_launch_without_any_token_keeps_the_order_of_its_neighbours(kernel):
    """With the overlap option on: a long kernel that releases its dependents early, a decode launch whose sequences are all
    empty, and a kernel that reads what the first one wrote."""
    c = Cache([0, 0, 0], 2, seed=92)
    q, out, qs, os_ = decode_case(c, 12, 0, 0, 0)
    ws = K.window_attention_workspace(3, c.mbps, 12, 2, weights=True)
    w = torch.zeros(c.blocks, 2, PAGE, device="cuda")
    rows, hidden = 100000, 1536
    x = torch.randn(rows, hidden, generator=c.g, device="cuda").half()
    gain = torch.ones(hidden, dtype=torch.float16, device="cuda")
    mid, last = torch.zeros_like(x), torch.zeros_like(x)

    def go():
        K.launch_rms_norm(mid, x, gain, rows, hidden, 1e-6)
        if kernel == "full":
            K.launch_paged_attention_decode(out, os_, q, qs, c.pool, c.tables, c.seq_lens, 3, c.mbps, 12, 2, D, SCALE)
        elif kernel == "window":
            K.launch_paged_window_attention_decode(out, os_, q, qs, c.pool, c.tables, c.seq_lens, 3, c.mbps, 12, 2, D, SCALE, 9, 0, ws)
        else:
            K.launch_paged_attention_decode_weights(out, os_, q, qs, c.pool, c.tables, c.seq_lens, 3, c.mbps, 12, 2, D, SCALE, w, ws)
        K.launch_rms_norm(last, mid, gain, rows, hidden, 1e-6)

    go()
    torch.cuda.synchronize()
    want = last.clone()
    K.set_attention_prologue_overlap(True)
    try:
        for _ in range(5):
            mid.zero_(), last.zero_()
            torch.cuda.synchronize()
            go()
            torch.cuda.synchronize()
            assert torch.equal(last, want)
    finally:
        K.set_attention_prologue_overlap(False)
    assert bool((out == 7.0).all())


def test_a_request_with_a_bounded_cache():
    """The operators as a serving loop uses them, against a 64-bit model of the same loop: a prompt ingested in two
    chunks with window attention, decode steps that scatter one token and accumulate weights, an eviction in place
    whenever the cache passes its budget, and window attention over what is left."""
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    kv, heads, budget, sinks, recent, window = 2, 12, 96, 4, 24, 40
    mbps, blocks = 20, 30
    order = (torch.randperm(blocks - 1, generator=g, device="cuda") + 1).int()
    table = order[:mbps].view(1, mbps).contiguous()
    pool = poison(blocks, 2, kv, PAGE, D).clone()
    w = torch.zeros(blocks, kv, PAGE, device="cuda")
    ws = K.window_attention_workspace(1, mbps, heads, kv, weights=True)
    model = [[[], [], []] for _ in range(kv)]              # per head: K rows, V rows, weights

    def append(k, v, at):
        n = k.shape[0]
        pos = torch.arange(at, at + n, device="cuda", dtype=torch.int32)
        K.launch_kv_scatter(pool, k.contiguous(), v.contiguous(), kv * D, kv * D, table, 0, pos, n, kv, D)
        for h in range(kv):
            model[h][0] += list(k.view(n, kv, D)[:, h].double())
            model[h][1] += list(v.view(n, kv, D)[:, h].double())
            model[h][2] += [0.0] * n

    def rnd(n, width):
        return torch.randn(n, width, generator=g, device="cuda").half()

    length = 0
    for rows in (70, 41):
        append(rnd(rows, kv * D), rnd(rows, kv * D), length)
        q = rnd(rows, heads * D)
        out = torch.empty_like(q)
        K.launch_paged_window_prefill_attention(out, heads * D, q, heads * D, pool, table, mbps, length, rows, heads, kv, D,
                                                SCALE, window, sinks, None)
        for i in (0, rows // 2, rows - 1):
            p = length + i
            t = torch.arange(p + 1, device="cuda")
            seen = (t < sinks) | (t > p - window)
            k = torch.stack([torch.stack(model[h][0][:p + 1]) for h in range(kv)])
            v = torch.stack([torch.stack(model[h][1][:p + 1]) for h in range(kv)])
            ref, tol, _, _ = attend64(q[i].double().view(kv, -1, D), k, v, seen)
            check(out[i].view(kv, -1, D), ref, tol, "prompt")
        length += rows
    lens = torch.zeros(1, dtype=torch.int32, device="cuda")
    evictions = 0
    for step in range(60):
        append(rnd(1, kv * D), rnd(1, kv * D), length)
        length += 1
        lens.fill_(length)
        q = rnd(1, heads * D)
        out, bounded = torch.empty_like(q), torch.empty_like(q)
        K.launch_paged_attention_decode_weights(out, heads * D, q, heads * D, pool, table, lens, 1, mbps, heads, kv, D, SCALE,
                                                w, ws)
        K.launch_paged_window_attention_decode(bounded, heads * D, q, heads * D, pool, table, lens, 1, mbps, heads, kv, D,
                                               SCALE, window, sinks, ws)
        k = torch.stack([torch.stack(model[h][0]) for h in range(kv)])
        v = torch.stack([torch.stack(model[h][1]) for h in range(kv)])
        every = torch.ones(length, dtype=torch.bool, device="cuda")
        ref, tol, p, _ = attend64(q[0].double().view(kv, -1, D), k, v, every)
        check(out[0].view(kv, -1, D), ref, tol, f"step {step}")
        t = torch.arange(length, device="cuda")
        ref, tol, _, _ = attend64(q[0].double().view(kv, -1, D), k, v, (t < sinks) | (t >= length - window))
        check(bounded[0].view(kv, -1, D), ref, tol, f"step {step}, window")
        for h in range(kv):
            got = p[h].sum(dim=0).tolist()
            model[h][2] = [a + b for a, b in zip(model[h][2], got)]
        if length > budget + 10 or step == 59:
            kept = torch.empty(1, kv, budget, dtype=torch.int32, device="cuda")
            K.launch_kv_evict(pool, w, table, mbps, table, mbps, lens, lens, kept, 1, kv, D, budget, sinks, recent)
            evictions += 1
            for h in range(kv):
                x = np.array(model[h][2])
                slots = kept[0, h].tolist()
                assert slots == sorted(set(slots)) and slots[:sinks] == list(range(sinks))
                assert slots[-recent:] == list(range(length - recent, length))
                rest = [j for j in range(sinks, length - recent)]
                dropped = [j for j in rest if j not in set(slots)]
                # what was dropped weighs no more than what stayed, up to the FP32 sums' error over the steps
                stayed = [j for j in rest if j in set(slots)]
                assert x[dropped].max() <= x[stayed].min() + 1e-5
                for part in range(3):
                    model[h][part] = [model[h][part][j] for j in slots]
            length = int(lens.item())
            assert length == budget
    assert evictions >= 5 and K.window_attention_health(ws) == 0
