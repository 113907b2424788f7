"""Edges of the paged K/V cache operators that the cases of test_paged_kv.py leave out; the cache, the reference in
float64 and its tolerance are that file's."""

import numpy as np
import pytest

from runtime import hb_lib
from test_paged_kv import Case, _torch, ints, tables

gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 6, 2 ** 40])
@pytest.mark.parametrize("heads,rows,lengths", [((14, 2, 64), [10, 3], [5, 70]), ((14, 2, 64), [300, 130], [200, 129]),
                                                ((16, 2, 128), [40, 300], [30, 500])])
def test_windows_wider_than_any_context(heads, rows, lengths, window):
    """They hide nothing, also in tiles whose first rows stand before the
    sequence (positions -5 .. -1 of the first case)."""
    torch = _torch()
    case = Case(heads, "bfloat16", rows, lengths, seed=41)
    plain, plain_lse = case.check()
    out, lse = case.check(window)
    assert torch.equal(out, plain) and torch.equal(lse, plain_lse)


def test_a_pool_in_host_memory_is_refused():
    """Before the library, or a device, is touched: the kernels would read host addresses."""
    torch = _torch()
    from runtime.paged_kv import PagedKVCache

    with pytest.raises(ValueError, match="CUDA"):
        PagedKVCache(1, 1, 64, 4, 2, 128, device="cpu")
    with pytest.raises(ValueError, match="CUDA"):
        PagedKVCache.wrap(torch.zeros((4, 1, 1, 2, 1, 64, 64), dtype=torch.bfloat16),
                          torch.zeros((2, 2), dtype=torch.int32), torch.zeros(4, dtype=torch.int32),
                          torch.zeros(2, dtype=torch.int32))


@gpu
@pytest.mark.parametrize("heads,rows", [((14, 2, 64), [2, 3, 1]), ((16, 2, 128), [200, 100, 50])])
def test_row_starts_that_descend_are_refused(heads, rows):
    """Entries would share rows, and their work could be any multiple of what
    the host has counted: the call gives zeros and says so, the next one runs."""
    torch = _torch()
    case = Case(heads, "bfloat16", rows, [250, 300, 270], seed=42)
    good, lse = case.check()
    a, b, c = np.cumsum(rows)
    right = case.row_start
    for bad in ([0, b, a, c], [0, a, c, b], [a, 0, b, c], [c, c, a, b]):
        case.row_start = ints(bad)
        out, none = case.attend(out=torch.full_like(case.q, 7.0))
        with pytest.raises(hb_lib.HbError, match="out of range"):
            case.cache.status()
        assert bool((out == 0).all()) and bool((none == -np.inf).all())
    case.row_start = right
    out, again = case.check()
    assert torch.equal(out, good) and torch.equal(again, lse)


@gpu
@pytest.mark.parametrize("heads,rows", [((14, 2, 64), [1, 0, 2]), ((14, 2, 64), [1, 1, 300]), ((16, 2, 128), [200, 200, 200])])
@pytest.mark.parametrize("before,after", [(0, 5), (3, 0), (2, 700)])
def test_rows_of_no_entry_give_zeros(heads, rows, before, after):
    """As a captured step with room for more rows has them; append gives q = 0 for the same rows."""
    torch = _torch()
    case = Case(heads, "bfloat16", rows, [250, 300, 400], seed=43)
    want, want_lse = case.check()
    n = case.n_rows
    shape = (before + n + after, case.qh, case.d)
    q = torch.randn(shape, device="cuda").to(case.dtype)
    q[before: before + n] = case.q
    case.q, case.row_start = q, case.row_start + before
    wide = torch.full((shape[0], case.qh, case.d + 1), 7.0, dtype=case.dtype, device="cuda")
    for out in (torch.full(shape, 7.0, dtype=case.dtype, device="cuda"), wide[:, :, 1:]):
        got, lse = case.attend(out=out)
        case.cache.status()
        assert torch.equal(got[before: before + n], want) and torch.equal(lse[before: before + n], want_lse)
        for part in (slice(0, before), slice(before + n, None)):
            assert bool((got[part] == 0).all()) and bool((lse[part] == -np.inf).all())
    assert bool((wide[:, :, 0] == 7).all())
    cos, sin = tables(case.d, 512)
    qkv = torch.randn((shape[0], (case.qh + 2 * case.kvh) * case.d), device="cuda").to(case.dtype)
    turned = case.cache.append(1, qkv, case.slots, case.row_start, case.max_rows, cos, sin)
    case.cache.status()
    assert not bool(turned[:before].any()) and not bool(turned[before + n:].any())


@gpu
@pytest.mark.parametrize("heads", [(14, 2, 64), (32, 2, 128)])
def test_mixed_steps_back_to_back(heads):
    """Steps that decode and prefill at once, each layer's append directly
    before its attention, nothing waited for: the same bits as when every
    call is waited for."""
    torch = _torch()
    from runtime.paged_kv import PagedKVCache

    qh, kvh, d = heads
    rows = [1, 260, 1, 90, 1]
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    qkv = torch.randn((12, sum(rows), (qh + 2 * kvh) * d), device="cuda", generator=g).bfloat16()
    cos, sin = tables(d, 4096)
    slots, start, counts = ints([3, 0, 4, 1, 2]), ints(np.concatenate([[0], np.cumsum(rows)])), ints(rows)

    def steps(wait):
        cache, outs = PagedKVCache(2, kvh, d, 120, 5, 2048), []
        q = torch.empty((sum(rows), qh, d), dtype=torch.bfloat16, device="cuda")
        for i in range(0, 12, 2):
            cache.reserve(slots, counts)
            for layer in range(2):
                cache.append(layer, qkv[i + layer], slots, start, max(rows), cos, sin, out=q)
                if wait:
                    torch.cuda.synchronize()
                outs.append(cache.attend(layer, q, slots, start, max(rows), lse=True))
                if wait:
                    torch.cuda.synchronize()
        cache.status()
        return outs

    want = steps(True)
    for _ in range(3):
        for (a, b), (c, e) in zip(steps(False), want):
            assert torch.equal(a, c) and torch.equal(b, e)
    # and captured, replayed back to back
    cache = PagedKVCache(1, kvh, d, 120, 5, 2048)
    cache.reserve(slots, counts)

    def layer():
        return cache.attend(0, cache.append(0, qkv[0], slots, start, max(rows), cos, sin), slots, start, max(rows), lse=True)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = layer()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = [layer() for _ in range(3)]
    for _ in range(20):
        graph.replay()
    cache.status()
    assert all(torch.equal(a, want[0]) and torch.equal(b, want[1]) for a, b in got)


@gpu
@pytest.mark.parametrize("heads", [(14, 2, 64), (32, 2, 128)])
def test_q_and_rope_tables_rewritten_between_calls_without_a_wait(heads):
    """The kernel before writes the tables that append turns by, append the q
    that attention reads, in the same memory each time."""
    torch = _torch()
    from runtime.paged_kv import PagedKVCache

    qh, kvh, d = heads
    n = 40
    g = torch.Generator(device="cuda")
    g.manual_seed(4)
    new = torch.randn((8, n, (qh + 2 * kvh) * d), device="cuda", generator=g).bfloat16()
    some = [tables(d, 1024)]
    for _ in range(7):
        some.append(tuple(t.roll(17, 0) for t in some[-1]))
    slots, start, ones = ints(range(n)), ints(range(n + 1)), ints([1] * n)

    def steps(wait):
        cache, outs = PagedKVCache(1, kvh, d, n * 8, n, 512), []
        cache.pool.fill_(0.5)
        cache.reserve(slots, ints([300 + i for i in range(n)]))
        q = torch.empty((n, qh, d), dtype=torch.bfloat16, device="cuda")
        qkv, cos, sin = torch.empty_like(new[0]), torch.empty_like(some[0][0]), torch.empty_like(some[0][1])
        for x, (c, s) in zip(new, some):
            cache.reserve(slots, ones)
            qkv.copy_(x)
            cos.copy_(c)
            sin.copy_(s)
            if wait:
                torch.cuda.synchronize()
            cache.append(0, qkv, slots, start, 1, cos, sin, out=q)
            if wait:
                torch.cuda.synchronize()
            outs.append(cache.attend(0, q, slots, start, 1, lse=True))
            if wait:
                torch.cuda.synchronize()
        cache.status()
        return outs

    want = steps(True)
    for _ in range(3):
        for (a, b), (c, e) in zip(steps(False), want):
            assert torch.equal(a, c) and torch.equal(b, e)


def poisoned(case, position, kind, value, dim=None):
    """Sets a position's K (0) or V (1) of the first entry, all dims of it or one."""
    page = case.cache.pool[int(case.table_np[case.slots_np[0], position // 64]), 1, :, kind, :, position % 64]
    if dim is None:
        page[:] = value
    else:  # 16-byte blocks lie at block ^ (position & 7)
        page[:, dim // 64, (dim % 64 // 8 ^ position % 8) * 8 + dim % 8] = value


def timed(call):
    torch = _torch()
    call()
    best = 1e9
    for _ in range(3):
        a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        a.record()
        call()
        b.record()
        torch.cuda.synchronize()
        best = min(best, a.elapsed_time(b))
    return best


@gpu
@pytest.mark.parametrize("kind", [0, 1])
@pytest.mark.parametrize("heads,rows,lengths", [((14, 2, 64), [1500], [1500]), ((16, 2, 128), [700], [900]),
                                                ((14, 2, 64), [1] * 8, [3000] * 8)])
def test_a_nan_that_rows_see_is_not_looked_for_again(heads, rows, lengths, kind):
    """Rows that see it are NaN from the first pass on; only rows that it is
    hidden from are done again."""
    torch = _torch()
    case = Case(heads, "bfloat16", rows, lengths, seed=44)
    clean, clean_lse = case.check()
    fast = timed(case.attend)
    poisoned(case, 3, kind, float("nan"))
    out, lse = case.attend()
    slow = timed(case.attend)
    case.cache.status()
    sees = torch.arange(lengths[0] - rows[0], lengths[0], device="cuda") >= 3
    n = rows[0]
    assert bool(torch.isnan(out[:n][sees]).all()) and bool(torch.isfinite(out[:n][~sees]).all())
    assert torch.equal(torch.isnan(lse[:n]), (sees & (kind == 0))[:, None].expand(n, case.qh))
    _, _, tol, _ = case.reference()
    assert bool(((out[:n][~sees].double() - clean[:n][~sees].double()).abs() <= 2 * tol[:n][~sees]).all())
    assert torch.equal(out[n:], clean[n:]) and torch.equal(lse[n:], clean_lse[n:])
    assert slow < 10 * fast + 0.5  # ms; a second pass over every row took hundreds of times as long


@gpu
def test_an_infinity_in_one_dim_of_v_stays_there():
    torch = _torch()
    case = Case((14, 2, 64), "bfloat16", [200, 5], [300, 90], seed=45)
    clean, lse = case.check()
    poisoned(case, 150, 1, float("inf"), dim=37)
    out, same = case.attend()
    case.cache.status()
    sees = torch.arange(100, 300, device="cuda") >= 150
    assert bool((out[:200][sees][:, :, 37] == np.inf).all()) and torch.equal(lse, same)
    out[:200, :, 37] = torch.where(sees[:, None], 0, out[:200, :, 37])
    clean[:200, :, 37] = torch.where(sees[:, None], 0, clean[:200, :, 37])
    _, _, tol, _ = case.reference()
    assert bool(((out.double() - clean.double()).abs() <= 2 * tol).all())


@gpu
@pytest.mark.parametrize("rows", [300, 1])
@pytest.mark.parametrize("where", ["K seen", "V seen", "hidden"])
def test_a_nan_in_a_long_context_leaves_the_status_clean(rows, where):
    """Rows are done again after the pipeline's last wait, not between waits
    with a limit."""
    torch = _torch()
    length = 160_000
    case = Case((4, 1, 64), "bfloat16", [rows, 1], [length, 64], seed=46)
    clean, _ = case.check()
    _, _, tol, _ = case.reference()
    poisoned(case, length - 1 if where == "hidden" else 5, 0 if where == "K seen" else 1, float("nan"))
    out, lse = case.attend()
    case.cache.status()
    nan = slice(rows - 1, rows) if where == "hidden" else slice(0, rows)
    assert bool(torch.isnan(out[nan]).all())
    fine = [i for i in range(rows + 1) if not nan.start <= i < nan.stop]
    assert bool(((out[fine].double() - clean[fine].double()).abs() <= 2 * tol[fine]).all())


@gpu
def test_layers_past_32_bits_are_refused():
    """2^32 + 1 is not layer 1."""
    torch = _torch()
    case = Case((4, 2, 64), "bfloat16", [1, 2], [5, 9], seed=47)
    cos, sin = tables(64, 64)
    qkv = torch.zeros((3, 8 * 64), dtype=torch.bfloat16, device="cuda")
    for layer in (2 ** 32 + 1, 2 ** 32, -2 ** 32, 2 ** 70):
        with pytest.raises(ValueError):
            case.cache.attend(layer, case.q, case.slots, case.row_start, 2)
        with pytest.raises(ValueError):
            case.cache.append(layer, qkv, case.slots, case.row_start, 2, cos, sin)


@gpu
def test_rows_of_missing_pages_are_refused():
    """rows() has no page to read there, and reads no other one's."""
    case = Case((4, 2, 64), "bfloat16", [1, 1], [200, 9], seed=48)
    slot = int(case.slots_np[0])
    assert case.cache.rows(1, slot).shape == (2, 2, 200, 64)
    for bad in (-1, 10 ** 6):
        case.cache.table[slot, 1] = bad
        with pytest.raises(ValueError):
            case.cache.rows(1, slot)
    case.cache.lengths[slot] = 10 ** 6
    with pytest.raises(ValueError):
        case.cache.rows(1, slot)


@gpu
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("heads", [(4, 4, 64), (3, 3, 128)])
def test_few_rows_keep_the_weights_low_halves(heads, dtype):
    """V chosen so that each output nearly cancels: what the weights lose in
    the product with V is then all there is to see.  The bound is
    test_paged_kv.py's with the weights' error as two halves have it: u^2 A,
    and in FP16 2^-25 of each |v| where the low half is below the normal range
    (the sum of the weights is at least 1)."""
    torch = _torch()
    qh, kvh, d = heads
    case = Case(heads, dtype, [1] * 16, [3] * 16, seed=49)
    case.q *= 0.25
    u = 2.0 ** -8 if dtype == "bfloat16" else 2.0 ** -11
    pool = case.cache.pool
    at = torch.arange(8, device="cuda")[None] ^ torch.arange(3, device="cuda")[:, None]  # [position, block]
    want, tol = [], []
    for b, slot in enumerate(case.slots_np):
        page = pool[int(case.table_np[slot, 0]), 1, :, :, :, :3].view(kvh, 2, d // 64, 3, 8, 8)
        index = at.view(1, 1, 1, 3, 8, 1).expand_as(page)
        plain = lambda: torch.take_along_dim(page, index, 4).transpose(2, 3).reshape(kvh, 2, 3, d).double()  # noqa: E731, B023
        k, v = plain().unbind(1)
        q = case.q[b].double()
        w = torch.softmax((k * q[:, None]).sum(-1) * d ** -0.5, 1)[..., None]
        v[:, 2] = -(w[:, :2] * v[:, :2]).sum(1) / w[:, 2]
        stored = v.to(case.dtype).reshape(kvh, 3, d // 64, 8, 8).transpose(1, 2)
        page[:, 1] = torch.take_along_dim(stored, index[:, 1], 3)
        v = plain()[:, 1]
        o, a = (w * v).sum(1), (w * v.abs()).sum(1)
        ds = (d + 8) * 2.0 ** -24 * (k.abs() * q[:, None].abs()).sum(-1).amax(1, keepdim=True) * d ** -0.5
        want.append(o)
        tol.append(u * o.abs() + (u * u + 2 * ds + 2.0 ** -18) * a + 2.0 ** -24
                   + (2.0 ** -25 * v.abs().sum(1) if dtype == "float16" else 0))
    out, _ = case.attend()
    case.cache.status()
    off = (out.double() - torch.stack(want)).abs() / torch.stack(tol)
    assert float(off.max()) <= 1, float(off.max())


def test_c_refusal_of_tables_past_32_bits():
    """Page counts of a call are summed in 32 bits: over all slots they can
    reach the table's entries."""
    import ctypes

    lib = hb_lib.load()
    fake = 1 << 20
    pool = dict(pages_dev=fake, page_stride=16384, n_pages=4, layers=1, kv_heads=1, head_dim=64, element=0,
                table_dev=fake, refs_dev=fake, lengths_dev=fake, workspace_dev=fake, workspace_bytes=1 << 60)
    make = lambda slots, width: ctypes.byref(hb_lib.HbPagePool(n_slots=slots, table_width=width, **pool))  # noqa: E731
    assert lib.hb_paged_workspace_bytes(make(1 << 10, 1 << 20)) > 0
    for slots, width in ((1 << 11, 1 << 20), (1 << 20, 1 << 12), (2 ** 31 - 1, 2)):
        assert lib.hb_paged_workspace_bytes(make(slots, width)) == 0
        assert lib.hb_pages_reserve(make(slots, width), 1, fake, fake, None) == hb_lib.HB_ERR_UNSUPPORTED


@gpu
@pytest.mark.parametrize("heads", [(14, 2, 64), (16, 2, 128)])
def test_rows_of_no_entry_where_one_kernel_has_all_entries(heads):
    """Entries alike, as max_rows says: whole chunks (201 x 3 rows of which 3
    belong to none), then single tokens (2 x 3, 3 of none), and starts that descend."""
    torch = _torch()
    for rows, most in (([200, 200, 200], 201), ([1, 1, 1], 2)):
        case = Case(heads, "bfloat16", rows, [250, 300, 400], seed=50)
        want, want_lse = case.check()
        n = case.n_rows
        case.q = torch.cat([torch.randn_like(case.q[:2]), case.q, torch.randn_like(case.q[:1])])
        case.row_start, case.max_rows = case.row_start + 2, most
        out, lse = case.attend(out=torch.full_like(case.q, 7.0))
        case.cache.status()
        assert torch.equal(out[2: n + 2], want) and torch.equal(lse[2: n + 2], want_lse)
        assert not bool(out[:2].any()) and not bool(out[-1].any())
        assert bool((lse[:2] == -np.inf).all()) and bool((lse[-1] == -np.inf).all())
        case.row_start = case.row_start[torch.tensor([0, 2, 1, 3], device="cuda")].contiguous()
        out, lse = case.attend(out=torch.full_like(case.q, 7.0))
        with pytest.raises(hb_lib.HbError, match="out of range"):
            case.cache.status()
        assert not bool(out.any()) and bool((lse == -np.inf).all())


@gpu
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("heads", [(14, 2, 64), (16, 2, 128)])
def test_an_infinity_in_v_reaches_a_single_token(heads, dtype):
    """Infinity in the dim that has it, whatever a weight's low half is; the other dims as without it."""
    torch = _torch()
    case = Case(heads, dtype, [1, 1], [300, 90], seed=51)
    clean, lse = case.check()
    poisoned(case, 150, 1, float("-inf"), dim=45)
    out, same = case.attend()
    case.cache.status()
    assert bool((out[0, :, 45] == -np.inf).all()) and torch.equal(lse, same) and torch.equal(out[1], clean[1])
    out[0, :, 45] = clean[0, :, 45]
    _, _, tol, _ = case.reference()
    tol[0, :, 45] = 1
    assert bool(((out.double() - clean.double()).abs() <= 2 * tol).all())
