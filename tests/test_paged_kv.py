"""The paged K/V cache operators (hb_paged_*, hb_pages_*, runtime/paged_kv.py)
against plain implementations: attention in float64, append bit for bit, the
page operators against books kept in Python.

Attention tolerance, per element of a row with weights w_j (float64) over the
positions it sees: the output is rounded once (u |o|, u = 2^-8 for BF16's 8
significant bits, 2^-11 for FP16's 11), the weights once (u A, A = sum w_j |v_j|; FP16 weights below its
normal range by 2^-25 each, on a scale that lets the largest weight be as
small as 2^-8), and FP32 scores are off by at most (head_dim + 8) 2^-24 S, S
the largest sum |q||k| scale, which moves a weight by twice that, relatively;
2^-18 A covers the FP32 sums and the exponential's last bits.
"""

import ctypes

import numpy as np
import pytest

from runtime import hb_lib

PAGE = 64
gpu = pytest.mark.gpu
HEADS = [(14, 2, 64), (9, 3, 64), (4, 4, 64), (32, 2, 128), (16, 1, 128), (1, 1, 64), (40, 1, 64)]


def _torch():
    import torch

    return torch


def ints(values):
    torch = _torch()
    return torch.tensor(np.asarray(values, np.int32), device="cuda")


def swizzle(x):
    """[..., 64, D] in plain order -> [..., D / 64, 64, 64] as pages store it, and back: the blocks change places in pairs."""
    torch = _torch()
    d = x.shape[-1]
    y = x.reshape(*x.shape[:-1], d // 64, 8, 8).movedim(-3, -4)  # [..., D / 64, 64, 8, 8]
    at = torch.arange(PAGE, device=x.device)[:, None]
    return y[..., at, torch.arange(8, device=x.device)[None] ^ (at & 7), :].reshape(*x.shape[:-2], d // 64, PAGE, 64)


class Case:
    """A cache of random K / V with shuffled pages, and the rows of a call."""

    def __init__(self, heads, dtype, rows, lengths, seed=0, layers=2, layer=1, extra=2, page_stride=None):
        torch = _torch()
        from runtime.paged_kv import PagedKVCache

        self.qh, self.kvh, self.d = heads
        self.dtype = getattr(torch, dtype)
        self.rows_of, self.len_of, self.layer = list(rows), list(lengths), layer
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        r = np.random.default_rng(seed)
        b = len(rows)
        n_slots = b + 1
        self.slots_np = r.permutation(n_slots)[:b]
        width = max(1, -(-max(max(lengths), 1) // PAGE)) + 1
        need = [-(-n // PAGE) for n in lengths]
        n_pages = sum(need) + extra
        order = r.permutation(n_pages)
        self.table_np = np.full((n_slots, width), -1, np.int64)
        at = 0
        for s, k in zip(self.slots_np, need):
            self.table_np[s, :k] = order[at: at + k]
            at += k
        lens = np.zeros(n_slots, np.int64)
        lens[self.slots_np] = lengths
        shape = (n_pages, layers, self.kvh, 2, self.d // 64, PAGE, 64)
        if page_stride is None:
            pool = torch.empty(shape, dtype=self.dtype, device="cuda")
        else:
            flat = torch.empty(page_stride * n_pages, dtype=self.dtype, device="cuda")
            inner = torch.empty(shape[1:], dtype=self.dtype, device="cuda").stride()
            pool = flat.as_strided(shape, (page_stride, *inner))
        for p in range(n_pages):
            pool[p].normal_(generator=g)
        self.cache = PagedKVCache.wrap(pool, ints(self.table_np), ints(np.bincount(
            self.table_np[self.table_np >= 0], minlength=n_pages)), ints(lens))
        self.slots, self.row_start = ints(self.slots_np), ints(np.concatenate([[0], np.cumsum(rows)]))
        self.n_rows, self.max_rows = int(sum(rows)), int(max(rows))
        self.q = torch.randn((self.n_rows, self.qh, self.d), device="cuda", generator=g).to(self.dtype)

    def attend(self, window=0, **more):
        return self.cache.attend(self.layer, self.q, self.slots, self.row_start, self.max_rows, window=window,
                                 lse=True, **more)

    def reference(self, window=0, scale=None):
        """(out, lse, tolerance of out, tolerance of lse) in float64, position by position of the table."""
        torch = _torch()
        scale = self.d ** -0.5 if scale is None else scale
        u = 2.0 ** -8 if self.dtype == torch.bfloat16 else 2.0 ** -11
        pool, group = self.cache.pool, self.qh // self.kvh
        table = self.cache.table.cpu().numpy()
        out = torch.zeros((self.n_rows, self.qh, self.d), dtype=torch.float64, device="cuda")
        lse = torch.full((self.n_rows, self.qh), -np.inf, dtype=torch.float64, device="cuda")
        tol, tol_lse = torch.zeros_like(out), torch.zeros_like(lse)
        at = 0
        for n, length, slot in zip(self.rows_of, self.len_of, self.slots_np):
            seen = [j for j in range(length) if 0 <= slot < table.shape[0] and j // PAGE < table.shape[1]
                    and 0 <= table[slot, j // PAGE] < pool.shape[0]]
            if n and seen:
                j = torch.tensor(seen, device="cuda")
                pages = torch.tensor(table[slot].astype(np.int64), device="cuda")[j // PAGE]
                # plain order: undo the swizzle position by position
                x = pool[pages, self.layer].reshape(len(seen), self.kvh, 2, self.d // 64, PAGE, 8, 8)
                x = x[torch.arange(len(seen), device="cuda"), :, :, :, j % PAGE]      # [seen, kvh, 2, d/64, 8, 8]
                block = (torch.arange(8, device="cuda")[None] ^ (j % 8)[:, None]).view(-1, 1, 1, 1, 8, 1)
                x = torch.take_along_dim(x, block, 4).reshape(len(seen), self.kvh, 2, self.d).double()
                pos = torch.arange(length - n, length, device="cuda")[:, None]
                hide = (j[None] > pos) | ((j[None] <= pos - window) if window else (j[None] < 0))
                for h in range(self.qh):
                    q = self.q[at: at + n, h].double()
                    k, v = x[:, h // group, 0], x[:, h // group, 1]
                    s = (q @ k.T * scale).masked_fill(hide, -np.inf)
                    some = ~hide.all(1)
                    w = torch.where(some[:, None], torch.softmax(s, 1), 0.0)
                    w = torch.where(hide, 0.0, w)
                    vis = v.clone()
                    o = w @ torch.nan_to_num(vis, nan=0.0, posinf=0.0, neginf=0.0)
                    a = w @ torch.nan_to_num(vis, nan=0.0, posinf=0.0, neginf=0.0).abs()
                    big = torch.where(hide, 0.0, (q.abs() @ k.abs().T * scale)).amax(1, keepdim=True)
                    ds = (self.d + 8) * 2.0 ** -24 * torch.nan_to_num(big, nan=0.0, posinf=0.0)
                    tail = len(seen) * 2.0 ** -17 if u < 2.0 ** -9 else 0.0
                    out[at: at + n, h] = o
                    lse[at: at + n, h] = torch.logsumexp(s, 1)
                    tol[at: at + n, h] = u * o.abs() + (u + 2 * ds + 2.0 ** -18) * a + 2.0 ** -8 * u * tail + 2.0 ** -24
                    tol_lse[at: at + n, h] = (ds + 2.0 ** -20 * (1 + lse[at: at + n, h].abs().nan_to_num(
                        nan=0.0, posinf=0.0)[:, None])).squeeze(1)
            at += n
        return out, lse, tol, tol_lse

    def check(self, window=0, got=None, scale=None):
        torch = _torch()
        out, lse = self.attend(window, **({} if scale is None else {"scale": scale})) if got is None else got
        self.cache.status()
        ref, ref_lse, tol, tol_lse = self.reference(window, scale)
        off = (out.double() - ref).abs()
        assert bool(torch.isfinite(out).all())
        assert bool((off <= tol).all()), f"off by {float((off / tol.clamp(min=1e-30)).max()):.3g} tolerances"
        none = ref_lse == -np.inf
        assert torch.equal(none, lse.double() == -np.inf)
        off = torch.where(none, 0.0, (lse.double() - ref_lse).abs())
        assert bool((off <= tol_lse)[~none].all()), f"lse off by {float(off.max()):.3g}"
        return out, lse


# ---- attention -----------------------------------------------------------------------
ROWS = {
    "tokens": ([1, 1, 1, 1, 1, 1], [1, 64, 65, 200, 0 + 63, 1000]),
    "chunks": ([1, 5, 64, 129, 0, 300], [1, 70, 64, 200, 17, 700]),
    "one long": ([1], [5000]),
    "late chunk": ([37], [3001]),
    "late long chunk": ([260, 3], [2500, 4]),
    "odd": ([2, 17, 31], [2, 1017, 127]),
}


@gpu
@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("rows", list(ROWS))
def test_attend_matches_float64(heads, rows):
    Case(heads, "bfloat16", *ROWS[rows], seed=len(rows)).check()


@gpu
@pytest.mark.parametrize("heads", [(14, 2, 64), (32, 8, 128)])
@pytest.mark.parametrize("rows", ["tokens", "chunks", "late long chunk"])
def test_attend_fp16(heads, rows):
    Case(heads, "float16", *ROWS[rows], seed=3).check()


@gpu
@pytest.mark.parametrize("window", [1, 7, 64, 65, 300, 100000])
@pytest.mark.parametrize("heads,rows", [((9, 3, 64), "chunks"), ((16, 2, 128), "late long chunk"),
                                        ((14, 2, 64), "tokens")])
def test_attend_window(heads, rows, window):
    Case(heads, "bfloat16", *ROWS[rows], seed=window).check(window)


@gpu
def test_attend_scale_and_steep_scores():
    """Scores up to hundreds: the running maximum moves far and weights vanish."""
    case = Case((14, 2, 64), "bfloat16", [1, 70, 200], [900, 333, 1500], seed=5)
    case.q *= 8
    case.check(scale=1.0)


@gpu
@pytest.mark.parametrize("heads", [(14, 2, 64), (16, 2, 128)])
def test_attend_rising_scores(heads):
    """Every page's scores top those before: each step rescales what it has."""
    torch = _torch()
    case = Case(heads, "bfloat16", [1, 140], [700, 900], seed=6)
    pool, d = case.cache.pool, case.d
    for s, n in zip(case.slots_np, case.len_of):
        for i in range(-(-n // PAGE)):
            k = torch.ones((case.kvh, PAGE, d), device="cuda") * (0.25 * i)
            pool[int(case.table_np[s, i]), 1, :, 0] = swizzle(k).to(case.dtype)
    case.q.fill_(1.0)
    case.check()


@gpu
@pytest.mark.parametrize("rows", [[1, 3, 2, 1], [40, 130, 20, 300]])
def test_rows_that_see_nothing(rows):
    """Positions before the sequence, no page, a page out of range, a slot
    out of range, a window whose pages were given up: zeros and -inf."""
    torch = _torch()
    lengths = [0, 2, 150, 700]
    case = Case((14, 2, 64), "bfloat16", rows, [max(1, x) for x in lengths], seed=7)
    case.len_of = lengths
    case.cache.lengths[torch.tensor(case.slots_np, device="cuda")] = ints(lengths)
    s = case.slots_np
    case.cache.table[int(s[2]), 1] = -1
    case.cache.table[int(s[2]), 0] = 10 ** 6
    case.cache.table[int(s[3]), :4] = -1
    out, lse = case.check()
    assert bool((out[: rows[0]] == 0).all())
    case.check(window=100)
    case.slots = case.slots.clone()
    case.slots[1] = 99
    case.len_of[1], case.slots_np = 0, np.array([s[0], 99, s[2], s[3]])
    case.check()


@gpu
def test_length_beyond_the_table():
    torch = _torch()
    case = Case((4, 2, 64), "bfloat16", [3, 150], [100, 300], seed=8)
    case.cache.lengths.fill_(2000)  # only the table's pages exist; past them nothing is mapped
    case.len_of = [2000, 2000]
    case.check()


@gpu
@pytest.mark.parametrize("heads", [(14, 2, 64), (16, 2, 128)])
@pytest.mark.parametrize("poison", [float("nan"), float("inf"), -float("inf"), "lowest"])
@pytest.mark.parametrize("rows", [[1, 1, 1], [5, 140, 300]])
def test_hidden_places_never_reach_a_row(heads, poison, rows):
    """Free pages, the rest of the last page, positions past a window and
    later rows' K and V hold infinities, NaN or the type's lowest value."""
    torch = _torch()
    lengths, window = [70, 333, 600], 50
    case = Case(heads, "bfloat16", rows, lengths, seed=9)
    p = torch.finfo(torch.bfloat16).min if poison == "lowest" else poison
    pool = case.cache.pool
    used = set(case.table_np[case.table_np >= 0].tolist())
    for page in range(pool.shape[0]):
        if page not in used:
            pool[page] = p
    pool[:, 0] = p  # the other layer
    for s, n, m in zip(case.slots_np, rows, lengths):
        pages = case.table_np[s]
        if m % PAGE:
            pool[int(pages[m // PAGE]), :, :, :, :, m % PAGE:] = p
        for j in range(max(0, m - n - window + 1)):
            if j % 7 == 0:
                pool[int(pages[j // PAGE]), 1, :, :, :, j % PAGE] = p
    case.check(window)


@gpu
@pytest.mark.parametrize("poison", [float("nan"), float("inf")])
def test_later_rows_never_reach_earlier_ones(poison):
    """The last position's K and V are poison: only the last row of the
    chunk may show it."""
    torch = _torch()
    for rows, length in ((5, 77), (200, 500)):
        case = Case((14, 2, 64), "bfloat16", [rows], [length], seed=10)
        page = int(case.table_np[case.slots_np[0], (length - 1) // PAGE])
        clean, _ = case.attend()
        case.cache.pool[page, 1, :, :, :, (length - 1) % PAGE] = poison
        out, lse = case.attend()
        assert not bool(torch.isfinite(out[-1]).all())
        off = (out[:-1].double() - clean[:-1].double()).abs()
        _, _, tol, _ = case.reference()
        assert bool((off <= 2 * tol[:-1]).all())  # both within their own
        assert bool(torch.isfinite(lse[:-1]).all())


@gpu
@pytest.mark.parametrize("rows,lengths", [([1, 1], [200, 70]), ([20, 150], [300, 150])])
def test_attend_strides_and_alignment(rows, lengths):
    """q and out as heads-first, and at odd element offsets."""
    torch = _torch()
    case = Case((6, 2, 64), "bfloat16", rows, lengths, seed=11)
    plain, lse = case.check()
    q = case.q
    case.q = q.transpose(0, 1).contiguous().transpose(0, 1)
    out = torch.empty((6, case.n_rows, 64), dtype=q.dtype, device="cuda").transpose(0, 1)
    got, _ = case.attend(out=out)
    assert torch.equal(got, plain) and got.data_ptr() == out.data_ptr()
    wide = torch.zeros((case.n_rows, 6, 67), dtype=q.dtype, device="cuda")
    wide[:, :, 1:65] = q
    case.q = wide[:, :, 1:65]
    room = torch.full((case.n_rows, 6, 65), 7.0, dtype=q.dtype, device="cuda")
    got, got_lse = case.attend(out=room[:, :, 1:])
    assert torch.equal(got, plain) and torch.equal(got_lse, lse) and bool((room[:, :, 0] == 7).all())


@gpu
@pytest.mark.parametrize("rows,length", [([1, 40], [500, 400]), ([200, 1], [900, 64])])
def test_pages_past_32_bit_offsets(rows, length):
    """Pages 512 MB apart: byte offsets pass 2^32 from the ninth page on."""
    torch = _torch()
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 24 GB")
    Case((14, 2, 64), "bfloat16", rows, length, seed=12, page_stride=1 << 28).check()


@gpu
def test_attend_repeats_bit_for_bit_and_on_another_stream():
    torch = _torch()
    case = Case((14, 2, 64), "bfloat16", [1] * 9 + [33, 300], list(range(100, 1000, 100)) + [2000, 3000], seed=13)
    a, la = case.check()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b, lb = case.attend()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(a, b) and torch.equal(la, lb)


@gpu
def test_attend_no_rows():
    case = Case((4, 2, 64), "bfloat16", [1, 0], [5, 9], seed=14)
    torch = _torch()
    empty = torch.empty((0, 4, 64), dtype=case.dtype, device="cuda")
    assert case.cache.attend(1, empty, ints([]), ints([0]), 0).shape == (0, 4, 64)
    assert case.cache.attend(1, empty, case.slots, ints([0, 0, 0]), 0).shape == (0, 4, 64)


@gpu
def test_a_captured_step_replays_with_new_lengths():
    """reserve, append and attend in a CUDA graph: each replay is the next
    position, its books moved on the device."""
    torch = _torch()
    from runtime.paged_kv import PagedKVCache

    qh, kvh, d = 6, 2, 64
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    cos, sin = tables(d, 256)
    steps = 80
    new = torch.randn((steps, 3, (qh + 2 * kvh) * d), device="cuda", generator=g).bfloat16()

    def build():
        cache = PagedKVCache(2, kvh, d, 12, 3, 256)
        return cache, ints([2, 0, 1]), ints([1, 1, 1]), ints([0, 1, 2, 3])

    def step(cache, slots, ones, start, qkv):
        cache.reserve(slots, ones)
        return [cache.attend(layer, cache.append(layer, qkv, slots, start, 1, cos, sin), slots, start, 1)
                for layer in range(2)]

    args = build()
    want = [[o.clone() for o in step(*args, new[i])] for i in range(steps)]
    args[0].status()
    args2 = build()
    qkv = new[0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*args2, qkv)
        args2[0].free(args2[1])
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(*args2, qkv)
    for i in range(steps):
        qkv.copy_(new[i])
        graph.replay()
        for a, b in zip(outs, want[i]):
            assert torch.equal(a, b), i
    args2[0].status()
    assert args2[0].lengths.tolist() == [steps] * 3


# ---- append --------------------------------------------------------------------------
def tables(d, positions):
    torch = _torch()
    inv = 1.0 / 1e4 ** (torch.arange(d // 2, device="cuda", dtype=torch.float32) / (d // 2))
    angle = torch.arange(positions, device="cuda", dtype=torch.float32)[:, None] * inv
    return torch.cos(angle).contiguous(), torch.sin(angle).contiguous()


def turned(x, cos, sin, pos):
    """rotate-half RoPE in FP32 with separate products, rounded once"""
    torch = _torch()
    h = x.shape[-1] // 2
    c, s = cos[pos][:, None], sin[pos][:, None]
    a, b = x[..., :h].float(), x[..., h:].float()
    return torch.cat([a * c - b * s, b * c + a * s], -1).to(x.dtype)


@gpu
@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("odd", [False, True])
def test_append_is_exact(heads, dtype, odd):
    torch = _torch()
    qh, kvh, d = heads
    rows, lengths = [1, 70, 0, 5, 129], [1, 100, 30, 64, 500]
    case = Case(heads, dtype, rows, lengths, seed=21)
    cos, sin = tables(d, 512)
    total, cols = sum(rows), (qh + 2 * kvh) * d
    pad = 3 if odd else 0  # an unaligned row stride and base
    store = torch.randn((total, cols + pad), device="cuda").to(case.dtype)
    qkv = store[:, pad: pad + cols]
    before = case.cache.pool.clone()
    q = case.cache.append(1, qkv, case.slots, case.row_start, case.max_rows, cos, sin)
    case.cache.status()
    pos = torch.cat([torch.arange(m - n, m) for n, m in zip(rows, lengths)]).cuda()
    x = qkv.reshape(total, qh + 2 * kvh, d)
    assert torch.equal(q, turned(x[:, :qh], cos, sin, pos))
    k, v = turned(x[:, qh: qh + kvh], cos, sin, pos), x[:, qh + kvh:]
    at = 0
    for s, n, m in zip(case.slots_np, rows, lengths):
        got = case.cache.rows(1, int(s))
        assert torch.equal(got[0][:, m - n:], k[at: at + n].transpose(0, 1))
        assert torch.equal(got[1][:, m - n:], v[at: at + n].transpose(0, 1))
        at += n
    # nothing else moved: put the old values back where rows went
    changed = (case.cache.pool.view(torch.int16) != before.view(torch.int16)).any(-1).any(4)  # [page, layer, kvh, 2, position]
    assert not bool(changed[:, 0].any())
    assert int(changed.any(2).any(2).sum()) <= total


@gpu
def test_append_out_of_place_rows():
    """A row without a page is dropped, a row past the RoPE tables and one
    before its sequence give q = 0, and the status says what happened."""
    torch = _torch()
    case = Case((4, 2, 64), "bfloat16", [3, 2, 2], [130, 1, 300], seed=22)
    cos, sin = tables(64, 140)
    case.cache.table[int(case.slots_np[0]), 2] = -1  # positions 128, 129
    qkv = torch.randn((7, 8 * 64), device="cuda").bfloat16()
    before = case.cache.pool.clone()
    q = case.cache.append(1, qkv, case.slots, case.row_start, 3, cos, sin)
    with pytest.raises(hb_lib.HbError):
        case.cache.status()
    case.cache.status()  # cleared
    pos = torch.tensor([127, 128, 129, 0], device="cuda")
    want = turned(qkv.view(7, 8, 64)[[0, 1, 2, 4], :4], cos, sin, pos)
    assert torch.equal(q[[0, 1, 2, 4]], want)
    assert bool((q[[3, 5, 6]] == 0).all())  # position -1; positions 298, 299
    changed = (case.cache.pool != before).any(-1).any(4).any(3).any(2)  # [page, layer, position]
    assert int(changed.sum()) == 2  # position 127 of the first, 0 of the second


# ---- pages ---------------------------------------------------------------------------
class Books:
    """The page operators in plain Python."""

    def __init__(self, n_pages, n_slots, width):
        self.refs, self.lengths = [0] * n_pages, [0] * n_slots
        self.table = [[-1] * width for _ in range(n_slots)]
        self.pages = {}  # page -> [PAGE] contents

    def free_list(self):
        return [p for p, n in enumerate(self.refs) if n == 0]

    def reserve(self, slots, counts):
        snap, plan, need = list(self.refs), [], 0
        for s, c in zip(slots, counts):
            old, end = self.lengths[s], self.lengths[s] + c
            if end > len(self.table[s]) * PAGE:
                return False
            for i in range(old // PAGE, -(-end // PAGE)) if c else []:
                pg = self.table[s][i]
                if pg < 0 or snap[pg] > 1:
                    plan.append((s, i, pg, old))
                    need += 1
        free = self.free_list()
        if need > len(free):
            return False
        for (s, i, pg, old), fresh in zip(plan, free):
            self.table[s][i] = fresh
            self.refs[fresh] = 1
            if pg >= 0:
                self.refs[pg] -= 1
                if i == old // PAGE and old % PAGE:
                    self.pages[fresh] = self.pages[pg][: old % PAGE] + self.pages[fresh][old % PAGE:]
        for s, c in zip(slots, counts):
            self.lengths[s] += c
        return True

    def fork(self, src, dst, counts):
        rows, free = [], self.free_list()
        if sum(1 for c in counts if c % PAGE) > len(free):
            return False
        for a, c in zip(src, counts):
            row = self.table[a][: c // PAGE]
            if c % PAGE:
                fresh, old = free.pop(0), self.table[a][c // PAGE]
                rows.append((row, fresh, old, c % PAGE))
            else:
                rows.append((row, -1, -1, 0))
        old_rows = [list(self.table[d]) for d in dst]
        for (row, fresh, old, held), d, c, gone in zip(rows, dst, counts, old_rows):
            now = row + ([fresh] if fresh >= 0 else [])
            self.table[d] = now + [-1] * (len(self.table[d]) - len(now))
            self.lengths[d] = c
            for p in now:
                self.refs[p] += 1
            for p in gone:
                if p >= 0:
                    self.refs[p] -= 1
            if fresh >= 0:
                self.pages[fresh] = self.pages[old][:held] + self.pages[fresh][held:]
        return True

    def free(self, slots):
        for s in slots:
            for p in self.table[s]:
                if p >= 0:
                    self.refs[p] -= 1
            self.table[s] = [-1] * len(self.table[s])
            self.lengths[s] = 0

    def compact(self):
        live = sum(n > 0 for n in self.refs)
        holes = [p for p in range(live) if self.refs[p] == 0]
        new = [p if n > 0 else -1 for p, n in enumerate(self.refs)]
        for p in range(live, len(self.refs)):
            if self.refs[p] > 0:
                to = holes.pop(0)
                new[p], self.refs[to], self.refs[p] = to, self.refs[p], 0
                self.pages[to] = list(self.pages[p])
        self.table = [[new[p] if p >= 0 else -1 for p in row] for row in self.table]
        return new


def same(cache, books):
    """The books agree, and each position of each page holds its number (every
    element of a position, in every layer and head, is the same)."""
    assert cache.table.tolist() == books.table
    assert cache.refs.tolist() == books.refs
    assert cache.lengths.tolist() == books.lengths
    pool = cache.pool
    assert bool((pool == pool[:, :1, :1, :1, :1, :, :1]).all())
    got = pool[:, 0, 0, 0, 0, :, 0].float().tolist()
    assert got == [books.pages[p] for p in range(pool.shape[0])]


def number(cache, books, slots, counts, r):
    """Writes numbers to the slots' last counts positions, on both sides."""
    for s, c in zip(slots, counts):
        for j in range(books.lengths[s] - c, books.lengths[s]):
            v = float(r.integers(0, 256))
            page = books.table[s][j // PAGE]
            assert books.refs[page] == 1  # what is written is the slot's own
            cache.pool[page, :, :, :, :, j % PAGE] = v
            books.pages[page][j % PAGE] = v


@gpu
@pytest.mark.parametrize("n_pages,n_slots,width,layers,heads,d", [(40, 9, 5, 3, 2, 64), (6000, 33, 7, 1, 1, 128),
                                                                  (13, 4, 4, 1, 3, 64), (6, 4, 4, 1, 1, 64)])
def test_page_operators_against_books(n_pages, n_slots, width, layers, heads, d):
    torch = _torch()
    from runtime.paged_kv import PagedKVCache

    r = np.random.default_rng(n_pages)
    cache = PagedKVCache(layers, heads, d, n_pages, n_slots, width * PAGE)
    books = Books(n_pages, n_slots, width)
    books.pages = {p: [0.0] * PAGE for p in range(n_pages)}
    refused = 0
    for turn in range(60):
        op = r.choice(["reserve", "reserve", "reserve", "fork", "free", "compact", "back"])
        n = int(r.integers(1, n_slots + 1))
        some = r.permutation(n_slots)[:n].tolist()
        ok = True
        if op == "reserve":
            counts = [min(int(r.integers(0, 100)), width * PAGE - books.lengths[s]) for s in some]
            ok = books.reserve(some, counts)
            cache.reserve(ints(some), ints(counts))
            if ok:
                number(cache, books, some, [min(c, 3) for c in counts], r)
        elif op == "fork":  # sources may be destinations: a permutation with repeats
            src = r.integers(0, n_slots, n).tolist()
            counts = [int(r.integers(0, books.lengths[s] + 1)) for s in src]
            ok = books.fork(src, some, counts)
            cache.fork(ints(src), ints(some), ints(counts))
        elif op == "free":
            some = some[: max(1, n // 3)]
            books.free(some)
            cache.free(ints(some + some[:1]))  # one of them named twice
        elif op == "compact":
            assert cache.compact().tolist() == books.compact()
        else:  # a rejected draft: lengths go back, pages stay
            for s in some:
                books.lengths[s] = max(0, books.lengths[s] - int(r.integers(0, 70)))
            cache.lengths.copy_(ints(books.lengths))
        if ok:
            cache.status()
        else:
            refused += 1
            with pytest.raises(hb_lib.HbError, match="exhausted"):
                cache.status()
        same(cache, books)
    assert n_pages > 6 or refused  # the smallest pool runs out


@gpu
def test_page_operators_refuse_on_the_device():
    """Slots out of range, a slot twice, lengths past the table, counts past
    the source: nothing changes, the status says so."""
    from runtime.paged_kv import PagedKVCache

    cache = PagedKVCache(1, 1, 64, 8, 3, 256)
    cache.reserve(ints([0, 2]), ints([70, 10]))
    cache.status()
    state = [t.tolist() for t in (cache.table, cache.refs, cache.lengths)]
    for call in (lambda: cache.reserve(ints([3]), ints([1])), lambda: cache.reserve(ints([-1]), ints([1])),
                 lambda: cache.reserve(ints([1, 1]), ints([1, 1])), lambda: cache.reserve(ints([0]), ints([200])),
                 lambda: cache.reserve(ints([0]), ints([-1])), lambda: cache.fork(ints([0]), ints([1]), ints([71])),
                 lambda: cache.fork(ints([0, 2]), ints([1, 1]), ints([1, 1])),
                 lambda: cache.fork(ints([5]), ints([1]), ints([0])),
                 lambda: cache.fork(ints([0]), ints([-2]), ints([0])), lambda: cache.free(ints([7])),
                 lambda: cache.copy_pages(ints([0]), ints([8])), lambda: cache.copy_pages(ints([-1]), ints([2]))):
        call()
        with pytest.raises(hb_lib.HbError, match="out of range"):
            cache.status()
        assert state == [t.tolist() for t in (cache.table, cache.refs, cache.lengths)]
    cache.reserve(ints([1]), ints([64]))  # and the slots are usable after it
    cache.status()
    assert cache.lengths.tolist() == [70, 64, 10]


@gpu
def test_append_after_an_exhausted_reserve_writes_nothing():
    torch = _torch()
    from runtime.paged_kv import PagedKVCache

    cache = PagedKVCache(1, 1, 64, 2, 2, 256)
    cache.reserve(ints([0]), ints([64]))
    cos, sin = tables(64, 256)
    qkv = torch.ones((100, 3 * 64), dtype=torch.bfloat16, device="cuda")
    cache.append(0, qkv[:64], ints([0]), ints([0, 64]), 64, cos, sin)
    before = cache.pool.clone()
    cache.reserve(ints([0]), ints([100]))  # needs two pages, one is free
    cache.append(0, 2 * qkv, ints([0]), ints([0, 100]), 100, cos, sin)
    assert torch.equal(cache.pool, before)
    with pytest.raises(hb_lib.HbError, match="exhausted"):
        cache.status()


@gpu
@pytest.mark.parametrize("heads", [(14, 2, 64), (32, 2, 128)])
def test_lists_rewritten_between_calls_without_a_wait(heads):
    """Slots, row starts and lengths that kernels of the same stream write
    directly before each call, for calls that decode and prefill at once: the
    same bits as when every call is waited for."""
    torch = _torch()
    from runtime.paged_kv import PagedKVCache

    qh, kvh, d = heads
    rows = [1, 300, 1, 77, 1, 2]
    n, total = len(rows), sum(rows)
    cache = PagedKVCache(1, kvh, d, 300, 12, 1500)
    cache.pool.normal_()
    q = torch.randn((total, qh, d), device="cuda").to(cache.dtype)
    cache.reserve(ints(range(12)), ints([900 + 37 * i for i in range(12)]))
    cache.status()
    r = np.random.default_rng(3)
    calls = []
    for _ in range(12):
        order = r.permutation(n)
        calls.append((ints(r.permutation(12)[:n]), ints(np.concatenate([[0], np.cumsum(np.asarray(rows)[order])])),
                      ints(r.integers(310, 900, 12))))
    slots, starts = torch.empty_like(calls[0][0]), torch.empty_like(calls[0][1])

    def call(x, wait):
        slots.copy_(x[0])
        starts.copy_(x[1])
        cache.lengths.copy_(x[2])
        if wait:
            torch.cuda.synchronize()
        out = cache.attend(0, q, slots, starts, max(rows), lse=True)
        if wait:
            torch.cuda.synchronize()
        return out

    want = [call(x, True) for x in calls]
    for _ in range(3):
        torch.cuda.synchronize()
        for (a, b), (c, e) in zip([call(x, False) for x in calls], want):
            assert torch.equal(a, c) and torch.equal(b, e)
    cache.status()


@gpu
@pytest.mark.parametrize("refused", ["past the table", "slot twice", "fork past the source"])
def test_append_after_a_refused_call_writes_nothing(refused):
    """Lengths stayed as they were, so the rows' positions would be those of
    rows that the slot holds already."""
    torch = _torch()
    from runtime.paged_kv import PagedKVCache

    cache = PagedKVCache(1, 1, 64, 8, 2, 256)
    cache.reserve(ints([0, 1]), ints([200, 20]))
    cos, sin = tables(64, 256)
    qkv = torch.ones((200, 3 * 64), dtype=torch.bfloat16, device="cuda")
    cache.append(0, qkv, ints([0]), ints([0, 200]), 200, cos, sin)
    before = cache.pool.clone()
    if refused == "past the table":
        cache.reserve(ints([0]), ints([60]))
    elif refused == "slot twice":
        cache.reserve(ints([0, 0]), ints([5, 5]))
    else:
        cache.fork(ints([1]), ints([0]), ints([21]))
    cache.append(0, 2 * qkv[:60], ints([0]), ints([0, 60]), 60, cos, sin)
    assert torch.equal(cache.pool, before)
    with pytest.raises(hb_lib.HbError, match="out of range"):
        cache.status()
    cache.reserve(ints([0]), ints([5]))  # usable again once the status is read
    cache.append(0, 2 * qkv[:5], ints([0]), ints([0, 5]), 5, cos, sin)
    cache.status()
    assert not torch.equal(cache.pool, before)


def test_c_refusals_of_sizes_past_32_bits():
    lib = hb_lib.load()
    fake = 1 << 20
    pool = ctypes.byref(hb_lib.HbPagePool(
        pages_dev=fake, page_stride=16384, n_pages=4, layers=1, kv_heads=1, head_dim=64, element=0, n_slots=2,
        table_width=1, table_dev=fake, refs_dev=fake, lengths_dev=fake, workspace_dev=fake, workspace_bytes=1 << 40))
    attend = lambda heads, rows: lib.hb_paged_attend(  # noqa: E731
        pool, 0, ctypes.byref(hb_lib.HbPagedRows(fake, fake, 1, rows, rows, 0)), ctypes.byref(hb_lib.HbPagedQuery(
            q_dev=fake, q_row_stride=0, q_head_stride=0, out_dev=fake, out_row_stride=0, out_head_stride=0, q_heads=heads,
            scale=1.0)), None)
    assert attend((1 << 16) + 1, 1) == hb_lib.HB_ERR_UNSUPPORTED
    assert attend(1 << 16, 1 << 15) == hb_lib.HB_ERR_UNSUPPORTED
    assert attend(1, (1 << 31) - 1) == hb_lib.HB_ERR_UNSUPPORTED
    assert lib.hb_paged_append(
        pool, 0, ctypes.byref(hb_lib.HbPagedRows(fake, fake, 1, 1, 1, 0)), ctypes.byref(hb_lib.HbPagedNew(
            qkv_dev=fake, qkv_row_stride=192, q_dev=fake, q_row_stride=64, q_head_stride=64, cos_dev=fake, sin_dev=fake,
            rope_positions=8, q_heads=1 << 28)), None) == hb_lib.HB_ERR_UNSUPPORTED


@gpu
def test_copy_pages_within_and_between_pools():
    torch = _torch()
    from runtime.paged_kv import PagedKVCache

    a, b = PagedKVCache(3, 2, 64, 9, 1, 64), PagedKVCache(3, 2, 64, 20, 1, 64)
    a.pool.normal_()
    was = a.pool.clone()
    a.copy_pages(ints([1, 8]), ints([0, 5]))
    a.copy_pages(ints([2, 3, 4]), ints([19, 0, 7]), to=b)
    a.copy_pages(ints([]), ints([]))
    a.status()
    assert torch.equal(a.pool[[0, 5]], was[[1, 8]]) and torch.equal(a.pool[[1, 2, 3, 4, 6, 7, 8]], was[[1, 2, 3, 4, 6, 7, 8]])
    assert torch.equal(b.pool[[19, 0, 7]], was[[2, 3, 4]]) and not bool(b.pool[[1, 2, 18]].any())


# ---- refusals ------------------------------------------------------------------------
@gpu
def test_python_refusals():
    torch = _torch()
    from runtime.paged_kv import PagedKVCache

    case = Case((4, 2, 64), "bfloat16", [1, 2], [5, 9], seed=31)
    cache, q = case.cache, case.q
    go = lambda **k: cache.attend(**{**dict(layer=1, q=q, slots=case.slots, row_start=case.row_start, max_rows=2), **k})  # noqa: E731
    cos, sin = tables(64, 64)
    qkv = torch.zeros((3, 8 * 64), dtype=torch.bfloat16, device="cuda")
    put = lambda **k: cache.append(**{**dict(layer=1, qkv=qkv, slots=case.slots, row_start=case.row_start,  # noqa: E731
                                             max_rows=2, cos=cos, sin=sin), **k})
    go(), put()
    for bad in (dict(layer=2), dict(layer=-1), dict(q=q.float()), dict(q=q[0]), dict(q=q[..., :32]), dict(q=q[:, :3]),
                dict(q=q.cpu()), dict(slots=case.slots.long()), dict(row_start=case.row_start[:2]),
                dict(row_start=case.row_start.float()), dict(max_rows=-1), dict(scale=0.0), dict(scale=-1.0),
                dict(scale=float("nan")), dict(window=-1), dict(out=q[:1]), dict(q=q.transpose(1, 2))):
        with pytest.raises(ValueError):
            go(**bad)
    for bad in (dict(layer=2), dict(qkv=qkv.float()), dict(qkv=qkv[:, :100]), dict(qkv=qkv[:, :192]), dict(cos=cos[:, :16]),
                dict(cos=cos.double()), dict(sin=sin[:10]), dict(slots=case.slots[:, None]), dict(out=q[:1])):
        with pytest.raises(ValueError):
            put(**bad)
    for bad in (lambda: cache.reserve(case.slots, case.slots[:1]), lambda: cache.reserve(ints([0] * 9), ints([0] * 9)),
                lambda: cache.fork(case.slots, case.slots[:1], case.slots), lambda: cache.free(case.slots.long()),
                lambda: cache.copy_pages(case.slots, case.slots[:1]),
                lambda: cache.copy_pages(case.slots, case.slots, to=PagedKVCache(1, 2, 64, 4, 1, 64)),
                lambda: PagedKVCache(1, 1, 80, 4, 1, 64), lambda: PagedKVCache(0, 1, 64, 4, 1, 64),
                lambda: PagedKVCache(1, 1, 64, 4, 1, 64, dtype=torch.float32),
                lambda: PagedKVCache.wrap(cache.pool, cache.table.long(), cache.refs, cache.lengths),
                lambda: PagedKVCache.wrap(cache.pool, cache.table, cache.refs[:-1], cache.lengths),
                lambda: PagedKVCache.wrap(cache.pool[..., :32], cache.table, cache.refs, cache.lengths)):
        with pytest.raises(ValueError):
            bad()


def test_c_refusals_without_a_device():
    """Every entry point checks its arguments before it touches a device."""
    lib = hb_lib.load()
    fake = 1 << 20
    pool = dict(pages_dev=fake, page_stride=16384, n_pages=4, layers=1, kv_heads=1, head_dim=64, element=0, n_slots=2,
                table_width=3, table_dev=fake, refs_dev=fake, lengths_dev=fake, workspace_dev=fake,
                workspace_bytes=1 << 40)
    make = lambda **k: ctypes.byref(hb_lib.HbPagePool(**{**pool, **k}))  # noqa: E731
    bad, unsupported = hb_lib.HB_ERR_INVALID_ARG, hb_lib.HB_ERR_UNSUPPORTED
    size = lib.hb_paged_workspace_bytes(make())
    assert 0 < size < 64 << 20
    assert lib.hb_paged_workspace_bytes(None) == 0
    assert lib.hb_paged_workspace_bytes(make(head_dim=96)) == 0
    rows = hb_lib.HbPagedRows(fake, fake, 1, 1, 1, 0)
    query = dict(q_dev=fake, q_row_stride=64, q_head_stride=64, out_dev=fake, out_row_stride=64, out_head_stride=64,
                 q_heads=1, scale=1.0)
    q = lambda **k: ctypes.byref(hb_lib.HbPagedQuery(**{**query, **k}))  # noqa: E731
    r = lambda **k: ctypes.byref(hb_lib.HbPagedRows(**{**dict(slots_dev=fake, row_start_dev=fake, entries=1, rows=1,  # noqa: E731
                                                              max_rows=1), **k}))
    att = lambda p, rr=None, qq=None, layer=0: lib.hb_paged_attend(p, layer, rr or ctypes.byref(rows), qq or q(), None)  # noqa: E731
    for want, p in ((bad, None), (unsupported, make(head_dim=32)), (unsupported, make(element=2)), (bad, make(n_pages=0)),
                    (bad, make(page_stride=16384 - 128)), (bad, make(page_stride=16384 + 64)), (bad, make(table_dev=None)),
                    (bad, make(pages_dev=fake + 64)), (bad, make(workspace_bytes=size - 1)), (bad, make(table_width=0)),
                    (bad, make(workspace_dev=fake + 128))):
        assert att(p) == want
        assert lib.hb_pages_free(p, 1, fake, None) == want
        assert lib.hb_paged_status(p, None, None) == want
    assert att(make(), layer=1) == bad and att(make(), layer=-1) == bad
    assert att(make(), rr=r(entries=-1)) == bad and att(make(), rr=r(slots_dev=None)) == bad
    assert att(make(), rr=r(entries=1025)) == unsupported
    for x in (dict(q_heads=0), dict(scale=0.0), dict(scale=float("nan")), dict(window=-1), dict(q_dev=None),
              dict(out_dev=fake + 1)):
        assert att(make(), qq=q(**x)) == bad
    assert att(make(kv_heads=2, page_stride=32768), qq=q(q_heads=3)) == bad
    assert lib.hb_paged_attend(make(), 0, None, q(), None) == bad
    assert lib.hb_paged_attend(make(), 0, r(), None, None) == bad
    assert att(make(), rr=r(rows=0)) == hb_lib.HB_OK  # nothing to do
    new = dict(qkv_dev=fake, qkv_row_stride=192, q_dev=fake, q_row_stride=64, q_head_stride=64, cos_dev=fake, sin_dev=fake,
               rope_positions=8, q_heads=1)
    app = lambda **k: lib.hb_paged_append(make(), 0, r(), ctypes.byref(hb_lib.HbPagedNew(**{**new, **k})), None)  # noqa: E731
    for x in (dict(qkv_dev=None), dict(q_dev=None), dict(cos_dev=fake + 4), dict(rope_positions=0), dict(q_heads=-1)):
        assert app(**x) == bad
    assert lib.hb_paged_append(make(), 0, r(), None, None) == bad
    for n in (-1, 3):
        assert lib.hb_pages_reserve(make(), n, fake, fake, None) == bad
        assert lib.hb_pages_fork(make(), n, fake, fake, fake, None) == bad
    assert lib.hb_pages_free(make(), -1, fake, None) == bad and lib.hb_pages_free(make(), 1, None, None) == bad
    assert lib.hb_pages_compact(make(), None, None) == bad
    assert lib.hb_pages_copy(make(), 1, fake, fake, fake + 8, 1, None) == bad
    assert lib.hb_pages_copy(make(), 1, fake, fake, fake, 0, None) == bad
    assert lib.hb_pages_copy(make(), 0, None, None, None, 0, None) == hb_lib.HB_OK
