"""Decisions that the engine and the attention mixer make on the host about a decode step: the classes of
sequence lengths that a decode graph is captured for, and the number of key ranges per sequence."""
from types import SimpleNamespace

import pytest

from quicknn_b200.engine.engine import Engine
from quicknn_b200.parts import MIXERS, PartSpec


def mixer(n_kv=4, head_dim=256, window=None, resident=296):
    pos = PartSpec("rotary", {"head_dim": head_dim, "theta": 1e4, "rotary_dim": head_dim})
    m = MIXERS.get("attention")(PartSpec("attention", {
        "hidden_size": 64, "n_heads": 2 * n_kv, "n_kv_heads": n_kv, "head_dim": head_dim, "scale": 0.1,
        "softcap": None, "window": window, "position": pos}))
    m._resident = resident
    return m


def step(n_seqs, longest, spread, max_seq=8192, tuning=None):
    return SimpleNamespace(n_seqs=n_seqs, longest=longest, spread=spread, max_seq=max_seq, tuning=tuning or {},
                           mode="decode")


def test_length_classes_are_coarse_and_bound_the_longest_sequence():
    assert Engine.length_classes([1]) == (256, 1.0)
    assert Engine.length_classes([256, 250]) == (256, 1.0)
    assert Engine.length_classes([257, 250]) == (512, 1.0)
    assert Engine.length_classes([8192] * 8) == (8192, 1.0)
    assert Engine.length_classes([2048, 1024, 1024, 1024]) == (2048, 1.6)       # 2048 / 1280
    assert Engine.length_classes([1000, 800, 700]) == (1024, 1.25)
    assert Engine.length_classes([4000] + [100] * 15) == (4096, 2.2)
    # a batch that decodes 300 tokens from prompts of 600..900 changes class once
    seen = {Engine.length_classes([600 + t, 750 + t, 900 + t]) for t in range(300)}
    assert len(seen) == 2


def test_key_ranges_at_equal_lengths_fill_whole_rounds_of_blocks():
    """What was measured at context 8192 with equal lengths: batch 1 takes 64 ranges, 8 nine, 12 six, 24 three (one
    round of blocks each); 28 sequences take five ranges (two rounds of 560 blocks on 296 places: faster than
    one round of two long ranges, while six ranges would need a third round)."""
    m = mixer()
    got = {b: m.decode_splits(step(b, 8192, 1.0)) for b in (1, 2, 4, 8, 12, 16, 24, 28, 32)}
    assert got == {1: 64, 2: 37, 4: 18, 8: 9, 12: 6, 16: 9, 24: 3, 28: 5, 32: 9}
    # all blocks fit the device at once up to 12 sequences and at 24
    assert all(got[b] * b * 4 <= 296 for b in (1, 2, 4, 8, 12, 24))
    # whole rounds: 16 x 4 x 9 = 576 blocks are two rounds of 296 places, 32 x 4 x 9 four
    assert -(-16 * 4 * 9 // 296) == 2 and -(-32 * 4 * 9 // 296) == 4
    assert {b: m.decode_splits(step(b, 2048, 1.0)) for b in (16, 32, 64)} == {16: 4, 32: 2, 64: 1}
    # a windowed layer sees at most its window
    assert mixer(window=4096).decode_splits(step(8, 8192, 1.0)) == 9
    assert mixer(window=128).decode_splits(step(8, 8192, 1.0)) == 4
    # short sequences: no range shorter than 32 keys
    assert m.decode_splits(step(1, 256, 1.0)) <= 8


def test_key_ranges_with_unequal_lengths_take_more_than_one_round():
    """64 sequences of very unequal lengths: one range each would let the longest set the pace; equal lengths
    at the same batch stay with few, long blocks."""
    m = mixer()
    assert m.decode_splits(step(64, 2048, 1.6)) == 4
    assert m.decode_splits(step(64, 2048, 1.0)) == 1
    assert m.decode_splits(step(32, 2048, 1.6)) == 4
    # the caller's fixed number wins
    assert m.decode_splits(step(64, 2048, 1.6, tuning={"decode_splits": 7})) == 7
    # lengths unknown (a step built by hand): the cache's longest sequence stands in
    assert m.decode_splits(step(8, 0, 0.0, max_seq=8192)) == 9


@pytest.mark.parametrize("n_kv,hd,resident", [(1, 64, 1184), (16, 128, 592), (8, 256, 296)])
def test_key_ranges_stay_within_what_the_kernels_take(n_kv, hd, resident):
    m = mixer(n_kv=n_kv, head_dim=hd, resident=resident)
    for b in (1, 3, 8, 40, 128, 256):
        for longest in (256, 1024, 8192):
            for spread in (1.0, 1.25, 1.6, 2.2):
                s = m.decode_splits(step(b, longest, spread))
                assert 1 <= s <= 64 and s <= max(1, longest // 32)


def test_rows_cut_off_a_prompt_product_only_where_a_round_of_tiles_is_saved():
    """The decision is a host function of the sizes: at the 2B layer sizes only the down product (inner size 9216),
    only just beyond a multiple of 2048 rows (72 -> 81 tiles of 256 x 256 on 74 pairs of SMs), and only up to 64 rows."""
    import torch
    from quicknn_b200.kernels import ops
    cpu = torch.device("cpu")                         # stands for 148 SMs
    down = lambda m: ops._rows_for_the_small_kernel(m, 2304, 9216, ops.EPI_NONE, cpu)            # noqa: E731
    assert [down(m) for m in (2048, 2049, 2112, 2113, 2304, 4096, 4097, 6145, 257, 100)] == [0, 1, 64, 0, 0, 0, 1, 1, 0, 0]
    for n_out, k, epi in ((4096, 2304, ops.EPI_NONE), (2304, 2048, ops.EPI_NONE), (9216, 2304, ops.EPI_GATED)):
        assert all(ops._rows_for_the_small_kernel(m, n_out, k, epi, cpu) == 0 for m in (2049, 4097, 6145, 8193))


def test_stages_of_decode_attention():
    """296 blocks at once with three stages, 444 with two.  Blocks of one length run in rounds: two rounds of 444 in the place of two of
    296 took up to 1.3 times as long.  Unequal lengths fill the device whatever the number."""
    from quicknn_b200.kernels.lib import load
    stages = load().qnn_attn_decode_stages
    sizes = (1, 296, 297, 444, 445, 512, 576, 592, 593, 888, 889, 1024, 1184, 1344, 3072)
    assert {n: stages(n, 296, 444, 0) for n in sizes} == {
        1: 3, 296: 3, 297: 2, 444: 2, 445: 3, 512: 3, 576: 3, 592: 3, 593: 2, 888: 2, 889: 2, 1024: 2, 1184: 2, 1344: 2, 3072: 2}
    assert {n: stages(n, 296, 444, 1) for n in sizes} == {n: 2 if n > 296 else 3 for n in sizes}
    assert stages(500, 0, 444, 1) == 3 and stages(500, 296, 0, 1) == 3     # a device that could not say


def test_a_decode_graph_knows_whether_its_lengths_are_uneven_where_the_kernel_asks():
    m = mixer()
    m.decode_splits = lambda step: 4
    assert m.schedule(step(18, 2048, 1.6)) == (4,)                          # one round of blocks
    assert m.schedule(step(28, 2048, 1.6)) == (4, True) and m.schedule(step(28, 2048, 1.0)) == (4, False)
    assert mixer(head_dim=128).schedule(step(128, 2048, 1.6)) == (mixer(head_dim=128).decode_splits(step(128, 2048, 1.6)),)
    w = mixer(window=256)
    w.decode_splits = m.decode_splits
    assert w.schedule(step(28, 1024, 1.6)) == (4, True) and w.schedule(step(28, 2048, 1.6)) == (4, False)      # nearly all beyond the window


def test_width_of_product_tiles_counts_the_writing_where_the_inner_size_is_short():
    from quicknn_b200.kernels.lib import load
    width, long_k = load().qnn_gemm_tcgen05_2cta_width, load().qnn_gemm_tcgen05_2cta_cols
    # widths that are no multiple of 128 write slowly: by the walk alone these took 192 columns and 4 to 15 % longer than with 256
    for M, N, K in ((8192, 2048, 512), (8192, 2048, 768), (8192, 3072, 512), (4096, 4096, 256)):
        assert long_k(M, N, 148) == 192 and width(M, N, K, 148) in (128, 256), (M, N, K)
    # measured best where the walk is long
    for (M, N, K), cols in {(256, 2304, 9216): 64, (640, 2304, 9216): 96, (1280, 2304, 9216): 192, (640, 4096, 2304): 192, (1280, 4096, 2304): 160,
                            (2048, 1536, 6144): 192, (2048, 2304, 9216): 256, (2048, 4096, 2304): 256}.items():
        assert width(M, N, K, 148) == cols, (M, N, K)
    assert all(width(M, N, K, 148) % 32 == 0 and 64 <= width(M, N, K, 148) <= 256 for M in (1, 129, 5000, 10 ** 6) for N in (8, 1000, 300000) for K in (8, 65, 70000))


def test_a_kernel_that_ran_nothing_is_not_reported_as_one_that_gave_up_waiting():
    from quicknn_b200.kernels.ops import wait_status_message
    assert "gave up waiting (status 5;" in wait_status_message(5) and "shared memory" not in wait_status_message(5)
    assert "shared memory" in wait_status_message(256) and "waiting" not in wait_status_message(256)
    both = wait_status_message(256 | 32)
    assert "gave up waiting (status 32;" in both and "shared memory" in both


def test_steps_whose_common_keys_go_to_different_kernels_do_not_share_a_graph(monkeypatch):
    """The division into ranges may be the same though one bound of the keys is for the kernel of few rows, the other for that of many."""
    import torch
    from quicknn_b200.engine.batch import StepSharing
    from quicknn_b200.kernels import ops
    monkeypatch.setattr(ops, "_sm_count", lambda device: 148)
    monkeypatch.setattr(ops, "shared_attention_pays", lambda *a: True)
    schedules, kernels = {}, {}
    for n_groups, rows in ((8, 32), (1, 128), (4, 64), (8, 16)):
        for n_kv, hd in ((4, 128), (8, 128), (4, 256), (2, 64)):
            m = mixer(n_kv=n_kv, head_dim=hd)
            for own in (128, 1024):
                for keys in (512, 1024, 2048, 4096, 8192, 16384):
                    sharing = StepSharing(n_groups, rows, keys, own)
                    s = step(n_groups * rows, 16384, 1.0)
                    s.sharing, s.act_dtype = sharing, torch.bfloat16
                    plan = m.shared_plan(s)
                    key = (n_groups, rows, n_kv, hd, m.schedule(s))
                    kernels.setdefault(key, set()).add(plan.kernels)
                    schedules.setdefault((n_groups, rows, n_kv, hd, plan[:2]), set()).add(plan.kernels)
    assert any(len(k) > 1 for k in schedules.values())               # equal divisions for different kernels do occur
    assert all(len(k) == 1 for k in kernels.values())


BF, FP = "bfloat16", "float32"
# heads, kv heads, head size, groups, rows of a group, positions that need not be read again, most common keys, most own keys; us with the common keys read
# once, and once per row: one B200, the plans of a step's bounds
MEASURED = [
    (BF, 8, 4, 256, 1, 128, 1040384, 8192, 100, 36.8, 483.7), (BF, 8, 4, 256, 1, 16, 3840, 256, 100, 9.7, 9.6),
    (BF, 16, 8, 256, 1, 8, 1344, 192, 100, 9.1, 9.0), (BF, 9, 1, 256, 1, 2, 1536, 1536, 100, 9.0, 9.2),
    (BF, 32, 16, 128, 1, 128, 1040384, 8192, 100, 48.0, 936.9), (BF, 32, 16, 128, 1, 8, 2688, 384, 100, 9.5, 8.9),
    (BF, 32, 16, 128, 1, 8, 3584, 512, 100, 9.6, 9.7), (BF, 32, 4, 128, 8, 4, 13248, 768, 100, 20.9, 14.8),
    (BF, 32, 4, 128, 4, 4, 14976, 1408, 100, 17.6, 13.8), (BF, 32, 4, 128, 1, 128, 1040384, 8192, 100, 38.2, 275.7),
    (BF, 32, 4, 128, 1, 16, 15360, 1024, 100, 12.6, 11.8), (BF, 8, 4, 128, 1, 32, 11904, 384, 100, 9.5, 8.6),
    (BF, 16, 1, 128, 4, 32, 63488, 704, 100, 29.6, 25.1), (BF, 16, 1, 128, 1, 128, 97536, 768, 100, 30.4, 27.4),
    (BF, 16, 1, 128, 4, 32, 732096, 7424, 100, 37.3, 133.2), (BF, 8, 4, 64, 1, 32, 11904, 384, 100, 8.6, 7.1),
    (BF, 8, 4, 64, 1, 32, 23808, 768, 100, 8.6, 8.9), (BF, 32, 8, 64, 1, 32, 23808, 768, 100, 18.3, 13.8),
    (BF, 32, 8, 64, 8, 4, 12288, 640, 100, 14.4, 12.0), (BF, 32, 8, 64, 1, 128, 1040384, 8192, 100, 32.9, 282.2),
    (BF, 32, 8, 64, 1, 32, 31744, 1024, 100, 16.4, 16.2), (BF, 16, 4, 64, 1, 128, 97536, 768, 100, 26.0, 21.8),
    (BF, 16, 4, 64, 1, 128, 1040384, 8192, 100, 35.5, 147.9), (BF, 8, 1, 64, 1, 128, 97536, 768, 100, 18.8, 12.4),
    (BF, 8, 1, 64, 16, 4, 83136, 1984, 1000, 18.6, 14.7), (BF, 12, 12, 64, 1, 2, 64, 64, 100, 4.7, 3.6),
    (FP, 6, 1, 24, 1, 128, 1040384, 8192, 100, 103.7, 372.0), (BF, 6, 2, 40, 1, 4, 768, 256, 1000, 11.3, 10.9),
    (BF, 6, 2, 40, 1, 128, 1040384, 8192, 100, 125.8, 443.6), (BF, 8, 2, 56, 1, 4, 1536, 512, 1000, 13.2, 12.6),
    (FP, 16, 2, 64, 1, 2, 8192, 8192, 100, 25.1, 18.6), (FP, 16, 2, 64, 1, 16, 3840, 256, 100, 15.1, 11.8),
    (FP, 16, 2, 64, 1, 8, 14336, 2048, 100, 17.6, 33.1), (FP, 8, 8, 16, 8, 4, 8256, 512, 1000, 39.9, 15.9),
    (FP, 8, 8, 16, 16, 4, 78336, 1984, 1000, 78.1, 47.3), (BF, 4, 4, 32, 16, 4, 38592, 1024, 1000, 37.1, 18.8),
    (FP, 4, 4, 32, 16, 4, 17472, 512, 1000, 47.2, 30.5), (FP, 4, 4, 32, 1, 128, 1040384, 8192, 100, 68.1, 282.2),
    (FP, 8, 8, 64, 8, 4, 8640, 512, 1000, 72.7, 42.0), (FP, 8, 8, 64, 1, 128, 1040384, 8192, 100, 179.7, 983.9),
    (FP, 8, 4, 64, 1, 16, 3840, 256, 100, 14.9, 9.8), (FP, 8, 4, 64, 16, 4, 10560, 256, 1000, 54.3, 43.8),
    (BF, 8, 8, 48, 8, 4, 8640, 512, 1000, 58.5, 29.4), (BF, 8, 8, 48, 1, 128, 1040384, 8192, 100, 146.9, 527.7),
    (BF, 8, 4, 96, 1, 16, 30720, 2048, 1000, 63.5, 37.2), (BF, 8, 4, 96, 1, 8, 14336, 2048, 1000, 37.4, 22.6),
    (BF, 8, 4, 96, 1, 32, 63488, 2048, 100, 50.0, 54.8), (BF, 8, 8, 80, 1, 32, 63488, 2048, 1000, 160.5, 94.0),
    (BF, 8, 8, 80, 1, 128, 1040384, 8192, 100, 341.2, 935.9), (FP, 8, 4, 256, 1, 16, 30720, 2048, 1000, 168.5, 111.4),
    (FP, 8, 4, 256, 1, 128, 1040384, 8192, 100, 807.8, 2047.8), (FP, 8, 2, 128, 1, 32, 63488, 2048, 1000, 87.1, 60.4),
    (BF, 16, 1, 320, 1, 8, 28672, 4096, 1000, 233.6, 118.1), (BF, 16, 1, 576, 1, 4, 6144, 2048, 1000, 135.9, 120.0),
    (BF, 8, 2, 512, 1, 128, 520192, 4096, 100, 1160.1, 779.0), (BF, 16, 1, 576, 1, 128, 520192, 4096, 100, 2398.8, 5122.9),
]


@pytest.mark.parametrize("case", MEASURED, ids=lambda c: "-".join(str(x) for x in c[:9]))
def test_common_keys_are_read_once_where_it_was_measured_to_pay(case):
    """Where the rule says once, that took at most 1.07 times as long; a gain of more than a third is not left.  (A step rounds the
    positions that are spared down by up to an eighth.)"""
    import torch
    from quicknn_b200.engine.batch import StepSharing
    from quicknn_b200.kernels import ops
    dtype, heads, n_kv, hd, groups, rows, spared, keys, own, once, per_row = case
    up = lambda n: 1 << max(n - 1, 0).bit_length()                          # noqa: E731
    for least in (spared, spared * 7 // 8 + 1):
        sharing = StepSharing(up(groups), up(rows), up(keys), up(own), spared=least)
        pays = ops.shared_attention_pays(getattr(torch, dtype), heads, n_kv, hd, sharing)
        if once > 1.07 * per_row:
            assert not pays
        if once < 0.66 * per_row:
            assert pays
    # without the number of spared positions the bounds say it; a user's own numbers may be exact
    exact = StepSharing(groups, rows, keys, own)
    assert ops.shared_attention_pays(getattr(torch, dtype), heads, n_kv, hd, exact) in (True, False)


def test_a_window_that_a_rows_own_keys_fill_leaves_nothing_to_share():
    import torch
    from quicknn_b200.engine.batch import StepSharing
    from quicknn_b200.kernels import ops
    bf = torch.bfloat16
    pays = lambda own, window: ops.shared_attention_pays(bf, 8, 4, 256, StepSharing(1, 8, 8192, own, spared=7 * 8000), window)      # noqa: E731
    assert pays(128, None) and pays(128, 4096) and pays(2048, 4096) and not pays(4096, 4096) and not pays(8192, 1024)
    assert not ops.shared_attention_pays(bf, 8, 4, 256, StepSharing(1, 1, 8192, 64, spared=0))
    assert not ops.shared_attention_pays(bf, 8, 4, 256, StepSharing(0, 0, 0, 64))


def test_a_step_counts_the_positions_that_need_not_be_read_again():
    """From the numbers as they are, rounded down by less than an eighth; the bounds are powers of two."""
    import torch
    from quicknn_b200.cache import KVCache
    from quicknn_b200.parts import CacheNeed
    cache = KVCache([CacheNeed(1, 4, None)], [None], 8192, 16, 2048, torch.float32, "cpu")
    eng = Engine.__new__(Engine)
    eng.cache = cache
    rows = []
    for n, copies in ((700, 4), (130, 2), (60, 1)):
        s = cache.allocate()
        cache.extend([(s, n)])
        mine = [s] + cache.fork([s] * (copies - 1))
        cache.extend([(x, n + 1 + 70 * i) for i, x in enumerate(mine)])
        rows += mine
    sharing, tables, row_group = eng._sharing(rows, [cache.length(s) for s in rows])
    assert (sharing.n_groups, sharing.rows, sharing.keys, sharing.own) == (2, 4, 1024, 512)
    true = 3 * 640 + 1 * 128                                                # whole pages of 700 and 130 positions
    assert true * 7 / 8 < sharing.spared <= true
    assert tables.tolist() == [0, 4, 0, 640, 4, 2, 0, 128] and row_group.tolist() == [0, 0, 0, 0, 1, 1, -1]
