"""Decode attention of rows that share pages, against the formula in 64 bits.

Cells that belong to no position hold NaN: what is read besides the keys that a row sees shows at once.  Tolerances, element by element, with
A = sum p |v| / sum p of the row: bfloat16 weights round by half a step, 2^-8 relative, so the sum is off by at most 2^-8 A; the fast tanh errs by
2^-11 of the score, which changes a weight by that factor; exponentials by less than 2^-20; the result rounds by 2^-8 of itself.  float32: a score
is a sum of hd products, off by at most (hd + 3) 2^-24 sum |q k|, which enters a weight and the sum of the weights; sums of n terms by n 2^-24."""
import numpy as np
import pytest
import torch

from quicknn_b200.kernels import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
PAGE = 64


class Batch:
    """groups: (begin, end, lengths of the rows); ``alone``: lengths of rows of no group; ``left_out``: rows without a sequence."""

    def __init__(self, groups, nq, nkv, hd, dtype, window=0, ring=0, alone=(), left_out=(), seed=0, extra_cols=0):
        g = torch.Generator(device=DEV).manual_seed(seed)
        rng = np.random.default_rng(seed)
        self.nq, self.nkv, self.hd, self.window, self.ring, self.dtype = nq, nkv, hd, window, ring, dtype
        self.lens = [n for _, _, ns in groups for n in ns] + list(alone)
        B = self.B = len(self.lens)
        self.row_group = [i for i, (_, _, ns) in enumerate(groups) for _ in ns] + [-1] * len(alone)
        row0 = np.cumsum([0] + [len(ns) for _, _, ns in groups])
        self.group_list = [(int(row0[i]), len(ns), a, e) for i, (a, e, ns) in enumerate(groups)]
        width = ring // PAGE if ring else max(1, max(-(-n // PAGE) for n in self.lens))
        n_pages = 1 + B * width
        order = rng.permutation(np.arange(1, n_pages))
        self.table = np.zeros((B + 2, width), dtype=np.int32)
        slots = rng.permutation(B + 2)[:B].astype(np.int32)          # the cache has more slots than the batch
        self.k_of, self.v_of = [], []
        self.k = torch.full((n_pages, nkv, PAGE, hd), float("nan"), device=DEV, dtype=dtype)
        self.v = torch.full_like(self.k, float("nan"))
        for b, n in enumerate(self.lens):
            kk, vv = (torch.randn((max(n, 1), nkv, hd), device=DEV, generator=g).to(dtype) for _ in range(2))
            pages = order[b * width:(b + 1) * width].copy()
            gi = self.row_group[b]
            if gi >= 0:
                r0, _, a, e = self.group_list[gi]
                if b != r0:                                          # positions a .. e - 1 as in the group's first row
                    e_ = min(e, n, self.lens[r0])
                    if e_ > a:
                        kk[a:e_], vv[a:e_] = self.k_of[r0][a:e_], self.v_of[r0][a:e_]
                    for p in range(a // PAGE, -(-e // PAGE)):
                        at = p % (ring // PAGE) if ring else p
                        if at < width and a <= p * PAGE and (p + 1) * PAGE <= e:
                            pages[at] = self.table[slots[r0], at]
            self.table[slots[b]] = pages
            self.k_of.append(kk)
            self.v_of.append(vv)
            pos = torch.arange(max(0, n - ring) if ring else 0, n, device=DEV)
            cell = pos % ring if ring else pos
            pg = torch.from_numpy(pages.astype(np.int64)).to(DEV)[cell // PAGE]
            self.k[pg, :, cell % PAGE] = kk[pos]
            self.v[pg, :, cell % PAGE] = vv[pos]
        wide = torch.randn((B, (nq + 2 * nkv) * hd + extra_cols), device=DEV, generator=g).to(dtype)
        self.qkv = wide[:, :(nq + 2 * nkv) * hd]
        self.slot_len = np.zeros(B + 2, dtype=np.int32)
        self.slot_len[slots] = self.lens
        self.slots = slots.copy()
        self.left_out = list(left_out)
        self.slots[self.left_out] = -1

    def i32(self, a):
        return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).to(DEV)

    def shared(self, keys=None):
        g = self.i32(np.asarray(self.group_list, dtype=np.int32).reshape(-1, 4))
        keys = keys or max([e - a for _, _, a, e in self.group_list] or [0])
        return ops.SharedKeys(g, self.i32(self.row_group), rows=max([r for _, r, _, _ in self.group_list] or [0]), keys=keys, own=max(self.lens))

    def run(self, scale, cap=None, ranges=None, slopes=None, sinks=None, keys=None):
        """``keys``: the bound of a group's keys that the call is told (it may take groups of many rows to another kernel)"""
        sh = self.shared(keys)
        plan = ops.shared_attention_plan(self.dtype, self.B, self.nq, self.nkv, self.hd, sh, self.window or None, ranges=ranges)
        scratch = torch.full((plan.scratch_bytes // 4,), float("nan"), device=DEV)
        return ops.attn_decode_shared(self.qkv, self.nq, self.nkv, self.hd, self.k, self.v, self.i32(self.table), PAGE, self.ring, self.i32(self.slots),
                                      self.i32(self.slot_len), sh, scale, cap, self.window or None, plan, scratch, slopes=slopes, sinks=sinks)

    def check(self, got, scale, cap=None, slopes=None, sinks=None, rows=None):
        nq, nkv, hd = self.nq, self.nkv, self.hd
        for b in rows if rows is not None else range(self.B):
            n = self.lens[b]
            if b in self.left_out or n == 0:
                assert not got[b].any(), b
                continue
            lo = max(0, n - self.window) if self.window else 0
            q = self.qkv[b, :nq * hd].double().view(nkv, nq // nkv, hd)
            k, v = self.k_of[b][lo:n].double(), self.v_of[b][lo:n].double()
            s = torch.einsum("khd,pkd->khp", q, k) * scale
            mag = torch.einsum("khd,pkd->khp", q.abs(), k.abs()) * scale
            if cap:
                s = cap * torch.tanh(s / cap)
            tops = s.abs().amax().item()
            if slopes is not None:
                d = torch.arange(n - 1 - lo, -1, -1, device=DEV, dtype=torch.float64)
                s = s - slopes.double().view(nkv, nq // nkv, 1) * d
                tops = max(tops, s.abs().amax().item())
            m = s.amax(-1, keepdim=True)
            p = torch.exp(s - m)
            total = p.sum(-1, keepdim=True)
            if sinks is not None:
                total = total + torch.exp(sinks.double().view(nkv, nq // nkv, 1) - m)
            want = torch.einsum("khp,pkd->khd", p / total, v).reshape(-1)
            size = torch.einsum("khp,pkd->khd", p / total, v.abs()).reshape(-1)
            if self.dtype == torch.bfloat16:
                # the exponent's own rounding in float32: |s| 2^-23 twice, beside the fast functions
                tol = (2.0 ** -8 + (2 * tops * 2.0 ** -11 if cap else 0) + (hd * mag.amax().item() + 4 * tops) * 2.0 ** -23 + 2.0 ** -19) * size + 2.0 ** -8 * want.abs()
            else:
                tol = (2 * ((hd + 3) * mag.amax().item() + 4 * tops) * 2.0 ** -24 + (2 * n + 30) * 2.0 ** -24) * size
            err = (got[b].double() - want).abs()
            assert (err <= tol + 1e-30).all(), (b, n, (err - tol).max().item(), err.max().item())


BF, FP = torch.bfloat16, torch.float32
HEADS = [(8, 4, 256, BF), (8, 4, 128, BF), (12, 2, 64, BF), (16, 1, 128, BF), (9, 1, 256, BF), (2, 1, 64, BF), (6, 1, 24, FP), (4, 2, 16, FP), (6, 3, 40, BF), (5, 5, 256, FP), (4, 1, 520, FP)]


@pytest.mark.parametrize("nq,nkv,hd,dtype", HEADS)
@pytest.mark.parametrize("cap", [None, 50.0])
def test_against_the_formula(nq, nkv, hd, dtype, cap):
    b = Batch([(0, 448, [449, 470, 512, 513]), (0, 128, [129, 200]), (0, 64, [64, 100, 65])], nq, nkv, hd, dtype, alone=[1, 77, 300, 0], seed=hd)
    b.check(b.run(hd ** -0.5, cap), hd ** -0.5, cap)


@pytest.mark.parametrize("rows", [1, 2, 3, 7, 8, 9, 17, 33, 70])
@pytest.mark.parametrize("nq,nkv,hd,dtype", [(8, 4, 256, BF), (4, 4, 128, BF), (16, 2, 64, BF), (6, 1, 24, FP)])
def test_rows_of_a_group(rows, nq, nkv, hd, dtype):
    lens = [640 + 1 + (37 * i) % 150 for i in range(rows)]
    b = Batch([(0, 640, lens)], nq, nkv, hd, dtype, seed=rows)
    b.check(b.run(hd ** -0.5, 30.0), hd ** -0.5, 30.0)


@pytest.mark.parametrize("nq,nkv,hd,dtype", [(4, 2, 64, BF), (6, 1, 24, FP)])
def test_batches_of_more_rows_than_are_asked_for_at_once(nq, nkv, hd, dtype):
    groups = [(0, 192, [193 + (i * 13) % 70 for i in range(n)]) for n in (140, 3, 20)]
    b = Batch(groups, nq, nkv, hd, dtype, alone=[50, 129], left_out=[0, 141, 163], seed=41)
    for keys in (None, 1 << 20):
        b.check(b.run(hd ** -0.5, 50.0, keys=keys), hd ** -0.5, 50.0)


@pytest.mark.parametrize("nq,nkv,hd,dtype", [(8, 2, 128, BF), (4, 4, 256, BF), (6, 1, 24, FP)])
@pytest.mark.parametrize("keys", [None, 1 << 20])
def test_groups_that_say_too_much(nq, nkv, hd, dtype, keys):
    # rows that the batch does not have, more rows than the launch was told of, a row whose group does not hold it, a group that is not there:
    # such rows read their keys themselves
    b = Batch([(0, 256, [300, 260, 270, 299, 301])], nq, nkv, hd, dtype, alone=[90], seed=43)
    want = b.run(hd ** -0.5)
    for groups, row_group, rows in (([(0, 99, 0, 256)], [0] * 5 + [-1], 8), ([(0, 5, 0, 256)], [0] * 5 + [-1], 3), ([(1, 3, 0, 256)], [0] * 6, 4),
                                    ([(-2, 4, 0, 256), (6, 2, 0, 256), (0, 2, 0, 256)], [2, 2, 0, 1, 7, -5], 4)):
        sh = ops.SharedKeys(b.i32(groups), b.i32(row_group), rows=rows, keys=keys or 256, own=301)
        plan = ops.shared_attention_plan(dtype, b.B, nq, nkv, hd, sh)
        scratch = torch.full((plan.scratch_bytes // 4,), float("nan"), device=DEV)
        got = ops.attn_decode_shared(b.qkv, nq, nkv, hd, b.k, b.v, b.i32(b.table), PAGE, 0, b.i32(b.slots), b.i32(b.slot_len), sh, hd ** -0.5, None, None, plan, scratch)
        b.check(got, hd ** -0.5)
    b.check(want, hd ** -0.5)


@pytest.mark.parametrize("pages", [1, 2, 3, 6, 7])
@pytest.mark.parametrize("nq,nkv,hd", [(8, 4, 256), (9, 1, 256), (8, 2, 128), (16, 2, 64)])
@pytest.mark.parametrize("cap", [None, 50.0, 90.0])
def test_many_rows(cap, nq, nkv, hd, pages):
    # more query rows than a warp holds: 128 at a time, one or two pages of the pairs there, all divisions of the pages
    rows = {256: 18, 128: 70, 64: 19}[hd]
    b = Batch([(0, pages * 64, [pages * 64 + 1 + i % 90 for i in range(rows)]), (64, 192, [200, 222])], nq, nkv, hd, BF, alone=[130], left_out=[3], seed=pages + hd)
    for ranges in ((1, 1), (2, 1), (3, 2), (9, 1)):
        for keys in (1, 1 << 20):                                    # by either kernel
            b.check(b.run(hd ** -0.5, cap, ranges, keys=keys), hd ** -0.5, cap)


@pytest.mark.parametrize("nq,nkv,hd", [(8, 4, 256), (8, 2, 128), (8, 1, 64)])
def test_many_rows_with_slopes_sinks_and_windows(nq, nkv, hd):
    g = torch.Generator(device=DEV).manual_seed(hd)
    slopes = torch.rand(nq, device=DEV, generator=g) * 0.02
    sinks = 3 * torch.randn(nq, device=DEV, generator=g)
    lens = [449 + 7 * i % 120 for i in range(34)]
    b = Batch([(0, 448, lens)], nq, nkv, hd, BF, seed=hd)
    for sl, si, cap in ((slopes, None, None), (slopes, sinks, 40.0), (None, sinks, 40.0)):
        b.check(b.run(hd ** -0.5, cap, (2, 2), slopes=sl, sinks=si, keys=1 << 20), hd ** -0.5, cap, sl, si)
    b = Batch([(0, 448, lens)], nq, nkv, hd, BF, window=300, seed=hd + 1)
    b.check(b.run(hd ** -0.5, None, (2, 1), keys=1 << 20), hd ** -0.5)
    b = Batch([(64 * 20, 64 * 24, [64 * 24 + 1 + i for i in range(60)])], nq, nkv, hd, BF, window=384, ring=384, seed=hd + 2)
    b.check(b.run(hd ** -0.5, 50.0, keys=1 << 20), hd ** -0.5, 50.0)


def test_many_rows_of_large_scores():
    b = Batch([(0, 704, [705 + i for i in range(40)])], 8, 4, 64, BF, seed=17)
    pages = torch.from_numpy(b.table[b.slots[0]].astype(np.int64)).to(DEV)
    pos = torch.arange(704, device=DEV)
    for sign in (1, -1):
        ramp = torch.linspace(-1, 1, 704, device=DEV) * sign
        keys = (b.qkv[0, :64].float() * 3 * ramp[:, None, None]).to(BF).expand(704, 4, 64)
        for k in b.k_of:
            k[:704] = keys
        b.k[pages[pos // 64], :, pos % 64] = keys
        for ranges in ((1, 1), (2, 1)):
            b.check(b.run(1.0, None, ranges, keys=1 << 20), 1.0)


@pytest.mark.parametrize("ranges", [(1, 1), (1, 3), (5, 1), (7, 4), (64, 40)])
@pytest.mark.parametrize("nq,nkv,hd,dtype", [(8, 4, 256, BF), (8, 2, 64, BF), (6, 1, 24, FP)])
def test_numbers_of_ranges(ranges, nq, nkv, hd, dtype):
    b = Batch([(0, 832, [840, 1001, 833]), (0, 0, [3, 90])], nq, nkv, hd, dtype, alone=[513], seed=sum(ranges))
    b.check(b.run(hd ** -0.5, None, ranges), hd ** -0.5)


@pytest.mark.parametrize("nq,nkv,hd,dtype", [(8, 4, 256, BF), (4, 2, 128, BF), (6, 1, 24, FP)])
@pytest.mark.parametrize("window", [1, 100, 256, 500])
def test_windows(window, nq, nkv, hd, dtype):
    # a window without a ring: rows see different parts of the common positions, some none of them
    b = Batch([(0, 512, [512, 520, 560, 700]), (64, 320, [321, 400]), (0, 256, [256, 100 + 256, 1000])], nq, nkv, hd, dtype, window=window, seed=window)
    b.check(b.run(hd ** -0.5, 50.0), hd ** -0.5, 50.0)


@pytest.mark.parametrize("nq,nkv,hd,dtype", [(8, 4, 256, BF), (4, 2, 64, BF), (6, 1, 24, FP)])
@pytest.mark.parametrize("window,ring", [(256, 256), (200, 256), (512, 512)])
def test_rings(window, ring, nq, nkv, hd, dtype):
    # rings that have wrapped: pages in front of the common ones hold a row's own newest keys beside older ones
    a, e = 1024 + 64, 1280
    if ring == 512:
        a = 1024 - 64
    b = Batch([(a, e, [1281, 1300, 1344 - 64 * (ring == 256)]), (0, 128, [130, 140])], nq, nkv, hd, dtype, window=window, ring=ring, alone=[ring, 2000, 5], seed=ring)
    b.check(b.run(hd ** -0.5, None), hd ** -0.5)


@pytest.mark.parametrize("nq,nkv,hd,dtype", [(8, 4, 256, BF), (8, 2, 128, BF), (6, 3, 16, FP)])
def test_slopes_and_sinks(nq, nkv, hd, dtype):
    g = torch.Generator(device=DEV).manual_seed(1)
    slopes = torch.rand(nq, device=DEV, generator=g) * 0.02
    sinks = 3 * torch.randn(nq, device=DEV, generator=g)
    b = Batch([(0, 384, [390, 450, 385, 511, 400])], nq, nkv, hd, dtype, alone=[33], seed=3)
    for sl, si in ((slopes, None), (None, sinks), (slopes, sinks)):
        b.check(b.run(hd ** -0.5, 20.0, slopes=sl, sinks=si), hd ** -0.5, 20.0, sl, si)


@pytest.mark.parametrize("nq,nkv,hd,dtype", [(8, 4, 256, BF), (4, 2, 64, BF), (6, 1, 24, FP)])
def test_rows_of_no_sequence_come_out_as_zeros(nq, nkv, hd, dtype):
    b = Batch([(0, 256, [300, 260, 270, 299]), (0, 64, [65, 66])], nq, nkv, hd, dtype, alone=[5], left_out=[0, 2, 4, 5, 6], seed=5)
    b.check(b.run(hd ** -0.5), hd ** -0.5)


@pytest.mark.parametrize("nq,nkv,hd,dtype", [(8, 4, 256, BF), (4, 2, 64, BF), (6, 1, 24, FP)])
def test_a_key_that_one_row_sees_stays_with_it(nq, nkv, hd, dtype):
    # position 100 of the common pages holds NaN and Inf; only the shorter row's window reaches it
    b = Batch([(0, 512, [513, 700, 690])], nq, nkv, hd, dtype, window=500, seed=9)
    page = int(b.table[b.slots[0], 1])
    b.k[page, :, 100 - 64] = float("nan")
    b.v[page, :, 100 - 64] = float("inf")
    got = b.run(hd ** -0.5)
    b.check(got, hd ** -0.5, rows=[1, 2])
    assert torch.isnan(got[0]).any()


def test_strided_rows_and_no_groups():
    b = Batch([(0, 128, [150, 180])], 8, 2, 128, BF, alone=[200, 64], seed=11, extra_cols=24)
    b.check(b.run(0.1, 50.0), 0.1, 50.0)
    b = Batch([], 8, 2, 128, BF, alone=[200, 64, 1], seed=12)
    b.check(b.run(0.1), 0.1)


def test_large_scores():
    # the reference of the exponentials has to rise many times, and fall from the first keys on
    b = Batch([(0, 640, [650, 700, 641])], 8, 4, 64, BF, seed=13)
    for sign in (1, -1):
        ramp = torch.linspace(-1, 1, 640, device=DEV) * sign
        for i in range(3):
            b.k_of[i][:640] = (b.qkv[0, :64].float() * 3 * ramp[:, None, None]).to(BF)
        pages = torch.from_numpy(b.table[b.slots[0]].astype(np.int64)).to(DEV)
        pos = torch.arange(640, device=DEV)
        b.k[pages[pos // 64], :, pos % 64] = b.k_of[0][:640]
        b.check(b.run(1.0), 1.0)


def test_same_bits_again_and_on_another_stream():
    b = Batch([(0, 1024, [1100, 1030, 1500]), (0, 512, [513, 600])], 8, 4, 256, BF, seed=21)
    one = b.run(0.06, 50.0)
    assert torch.equal(one, b.run(0.06, 50.0))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        two = b.run(0.06, 50.0)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(one, two)


def test_a_captured_call_reads_lengths_and_groups_when_it_runs():
    b = Batch([(0, 512, [513, 560, 600])], 8, 4, 256, BF, seed=22)
    sh = b.shared()
    plan = ops.shared_attention_plan(BF, b.B, 8, 4, 256, sh)
    scratch = torch.empty(plan.scratch_bytes, dtype=torch.uint8, device=DEV)
    table, slots, lens = b.i32(b.table), b.i32(b.slots), b.i32(b.slot_len)
    args = (b.qkv, 8, 4, 256, b.k, b.v, table, PAGE, 0, slots, lens, sh, 0.06, None, None, plan, scratch)
    ops.attn_decode_shared(*args)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = ops.attn_decode_shared(*args)
    for end, cut in ((512, 0), (448, 30), (0, 1), (512, 90)):
        sh.groups[0, 3] = end
        for i in range(3):
            lens[b.slots[i]] = b.lens[i] - cut
        g.replay()
        torch.cuda.synchronize()
        keep, b.lens = b.lens, [n - cut for n in b.lens]
        b.check(out, 0.06)
        b.lens = keep


@pytest.mark.parametrize("nq,nkv,hd,rows,keys", [(8, 4, 256, 3, None), (8, 4, 96, 3, None), (8, 4, 256, 20, 1 << 20)])
def test_pages_far_into_a_long_cache(nq, nkv, hd, rows, keys):
    """elements of the pools behind the 2^31st, by every kernel"""
    b = Batch([(0, 256, [300 + r for r in range(rows)])], nq, nkv, hd, BF, seed=24)
    off = (1 << 31) // (nkv * PAGE * hd) + 3
    far = []
    for pool in (b.k, b.v):
        t = torch.empty((off + pool.shape[0], nkv, PAGE, hd), device=DEV, dtype=BF)
        t[off:] = pool
        far.append(t)
    b.k, b.v = far
    b.table = np.where(b.table > 0, b.table + off, 0).astype(np.int32)
    b.check(b.run(0.06, None, keys=keys), 0.06)


def test_the_same_as_attention_that_shares_nothing():
    b = Batch([(0, 960, [961, 1000, 1111, 1400])], 8, 4, 256, BF, seed=23)
    got = b.run(0.0625, 50.0)
    splits = 4
    o, ml = torch.empty(b.B * 8 * splits * 256, device=DEV), torch.empty(b.B * 8 * splits * 2, device=DEV)
    want = ops.attn_decode(b.qkv, 8, 4, 256, b.k, b.v, b.i32(b.table), PAGE, 0, b.i32(b.slots), b.i32(b.slot_len), 0.0625, 50.0, None, splits, o, ml)
    # both within the bound of the formula; next to one another a rounding each
    assert ((got.double() - want.double()).norm() / want.double().norm()).item() < 8e-3


def test_refusals():
    b = Batch([(0, 128, [150, 180])], 8, 2, 64, BF, seed=31)
    sh = b.shared()
    plan = ops.shared_attention_plan(BF, 2, 8, 2, 64, sh)
    scratch = torch.empty(plan.scratch_bytes, dtype=torch.uint8, device=DEV)
    args = dict(qkv=b.qkv, n_heads=8, n_kv=2, head_dim=64, k_pool=b.k, v_pool=b.v, page_table=b.i32(b.table), page_size=PAGE, ring=0, slots=b.i32(b.slots),
                slot_len=b.i32(b.slot_len), shared=sh, scale=0.1, cap=None, window=None, plan=plan, scratch=scratch)
    ops.attn_decode_shared(**args)
    for change in (dict(n_kv=3), dict(head_dim=128), dict(page_size=32), dict(ring=128), dict(ring=128, window=200), dict(ring=100, window=64), dict(scratch=scratch[:-16]),
                   dict(slots=b.i32(b.slots)[:1]), dict(plan=ops.SharedPlan(plan.common_ranges + 1, plan.own_ranges, plan.scratch_bytes)),
                   dict(slot_len=b.i32(b.slot_len)[:-1]), dict(window=-1), dict(v_pool=b.v[:-1])):
        with pytest.raises((ValueError, ops._lib.KernelError)):
            ops.attn_decode_shared(**{**args, **change})
    with pytest.raises(TypeError):
        ops.attn_decode_shared(**{**args, "v_pool": b.v.float()})
    with pytest.raises(ValueError):
        ops.shared_attention_plan(BF, 2, 8, 2, 60, sh)
    with pytest.raises(ValueError):
        ops.shared_attention_plan(BF, 2, 8, 2, 64, sh, ranges=(0, 1))
    with pytest.raises(ValueError):
        ops.SharedKeys(sh.groups[:, :3].contiguous(), sh.row_group, rows=2, keys=1, own=1)
    with pytest.raises(ValueError):
        ops.SharedKeys(sh.groups, sh.row_group, rows=0, keys=1, own=1)


@pytest.mark.parametrize("nq,nkv,hd", [(8, 4, 256), (8, 2, 128), (16, 2, 64)])
@pytest.mark.parametrize("cap", [None, 50.0])
def test_many_rows_captured_behind_a_kernel_that_writes_their_queries(nq, nkv, hd, cap):
    """Two calls of the two-kernel form on one scratch, each behind a kernel of this library that writes its queries, replayed back to back
    with other lengths and groups: the kernel of the rows' own keys starts beside that of the common ones and must not be early."""
    b = Batch([(0, 512, [513 + 3 * i for i in range(20)]), (0, 128, [150, 200, 129])], nq, nkv, hd, BF, alone=[70], seed=hd)
    B, sh = b.B, b.shared(keys=1 << 20)
    plan = ops.shared_attention_plan(BF, B, nq, nkv, hd, sh)
    assert plan.kernels == 3
    scratch = torch.full((plan.scratch_bytes // 4,), float("nan"), device=DEV)
    g = torch.Generator(device=DEV).manual_seed(1)
    rows = torch.randn((3 * B, b.qkv.shape[1]), device=DEV, generator=g).to(BF)          # rows 0 .. B - 1 are the step's
    table, slots, lens = b.i32(b.table), b.i32(b.slots), b.i32(b.slot_len)

    def call(k):
        ops.copy_slots([rows], list(range(k * B, (k + 1) * B)), list(range(B)))
        return ops.attn_decode_shared(rows[:B], nq, nkv, hd, b.k, b.v, table, PAGE, 0, slots, lens, sh, hd ** -0.5, cap, None, plan, scratch)

    call(1)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = [call(1), call(2)]
    whole, got = list(b.lens), []
    steps = ((512, 0), (448, 0), (0, 0), (512, 100), (512, 0))
    for end, cut in steps:                                           # nothing waits between the replays
        sh.groups[0, 3] = end
        lens[torch.from_numpy(b.slots[:20].astype(np.int64)).to(DEV)] = b.i32([n - cut for n in whole[:20]])
        graph.replay()
        got.append([o.clone() for o in outs])
    torch.cuda.synchronize()
    ops.raise_on_status(torch.device(DEV))
    for (end, cut), pair in zip(steps, got):
        b.lens = [n - cut for n in whole[:20]] + whole[20:]
        for k, o in enumerate(pair):
            b.qkv = rows[(k + 1) * B:(k + 2) * B]
            b.check(o, hd ** -0.5, cap)
    assert all(torch.equal(x, y) for x, y in zip(got[0], got[4]))


@pytest.mark.parametrize("nq,nkv,hd,dtype,keys", [(8, 4, 256, BF, 1 << 20), (8, 2, 128, BF, 1 << 20), (16, 2, 64, BF, 1 << 20), (8, 2, 128, BF, 1), (6, 1, 24, FP, 1)])
@pytest.mark.parametrize("cap", [None, 50.0])
def test_same_bits_whatever_ran_before(nq, nkv, hd, dtype, keys, cap):
    """results go by the numbers of ranges, not by what runs when or what the scratch holds"""
    b = Batch([(0, 640, [641 + 5 * i for i in range(40)]), (0, 64, [90, 65])], nq, nkv, hd, dtype, alone=[300], seed=3)
    one = b.run(hd ** -0.5, cap, (3, 2), keys=keys)
    assert torch.isfinite(one).all()
    for _ in range(20):
        assert torch.equal(one, b.run(hd ** -0.5, cap, (3, 2), keys=keys))


@pytest.mark.parametrize("nq,nkv,hd,dtype,rows,keys", [(8, 4, 256, BF, 3, None), (8, 2, 128, BF, 3, None), (16, 2, 64, BF, 3, None), (8, 2, 128, BF, 40, 1 << 20), (6, 1, 24, FP, 3, None),
                                                       (4, 2, 96, BF, 3, None)])
@pytest.mark.parametrize("window", [0, 300])
def test_page_tables_for_millions_of_positions(nq, nkv, hd, dtype, rows, keys, window):
    """more page ids than fit beside the tiles"""
    b = Batch([(0, 448, [450 + 31 * r for r in range(rows)])], nq, nkv, hd, dtype, alone=[200], window=window, seed=hd)
    wide = np.zeros((b.table.shape[0], 60000), dtype=np.int32)
    wide[:, :b.table.shape[1]] = b.table
    b.table = wide
    b.check(b.run(hd ** -0.5, 50.0, keys=keys), hd ** -0.5, 50.0)


@pytest.mark.parametrize("nq,nkv,hd", [(8, 4, 256), (4, 2, 64)])
def test_rings_of_millions_of_positions(nq, nkv, hd):
    """of which sequences have filled little"""
    b = Batch([(0, 448, [450, 500, 700])], nq, nkv, hd, BF, window=60000 * 64, ring=0, seed=hd)
    wide = np.zeros((b.table.shape[0], 60000), dtype=np.int32)
    wide[:, :b.table.shape[1]] = b.table
    b.table, b.ring = wide, 60000 * 64
    b.check(b.run(hd ** -0.5), hd ** -0.5)
