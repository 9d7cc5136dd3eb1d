"""Host side of the linear layers on dense weights: how tiles are shared out, workspace sizes, refusals without a GPU."""
import ctypes
import random

import pytest


@pytest.mark.parametrize("workers", [148, 74, 1, 13])
@pytest.mark.parametrize("overhead", [-1, 0, 4, 20])
def test_plan_covers_every_k_block_once(sp, workers, overhead):
    rng = random.Random(workers * 100 + overhead)
    for tiles, kb in [(0, 5), (1, 1), (1, 300), (workers, 7), (workers + 1, 64), (2 * workers - 1, 3)] + \
            [(rng.randint(1, 500), rng.randint(1, 300)) for _ in range(30)]:
        pieces = {}
        for worker, segments in enumerate(sp.linear_plan(tiles, kb, workers, overhead)):
            # a worker parks at most one piece: it has one slot
            assert sum(first != last for _, _, _, first, last in segments) <= 1
            for tile, k0, k1, first, last in segments:
                assert 0 <= tile < tiles and 0 <= k0 < k1 <= kb
                pieces.setdefault(tile, []).append((k0, k1, worker, first, last))
        assert sorted(pieces) == list(range(tiles))
        counters = set()
        for parts in pieces.values():
            parts.sort()
            assert parts[0][0] == 0 and parts[-1][1] == kb and all(a[1] == b[0] for a, b in zip(parts, parts[1:]))
            owners = [p[2] for p in parts]
            assert owners == list(range(owners[0], owners[-1] + 1)) and len(owners) <= 16
            assert all(p[3] == owners[0] and p[4] == owners[-1] for p in parts)
            assert overhead >= 0 or len(parts) == 1
            if len(parts) > 1:  # arrivals are counted under the first owner
                assert owners[0] not in counters
                counters.add(owners[0])


def test_plan_evens_out_few_tiles(sp):
    """72 tiles of 72 k-blocks on 148 workers: two equal parts each."""
    plan = sp.linear_plan(72, 72, 148, 4)
    assert sorted(sum(s[2] - s[1] for s in segments) for segments in plan) == [0] * 4 + [36] * 144


def test_plan_cuts_only_where_it_pays(sp):
    whole = [(0, 0, 16, 0, 0)]
    assert sp.linear_plan(1, 16, 148, 17)[0] == whole  # 6 k-blocks and 17 of overhead are more than 16
    assert len([w for w in sp.linear_plan(1, 36, 148, 17) if w]) == 5  # 7 * 5 * 5 <= 5 * 36
    assert len([w for w in sp.linear_plan(1, 1000, 148, 17) if w]) == 16
    assert len([w for w in sp.linear_plan(1, 1000, 148, 17, 4) if w]) == 4
    assert sp.linear_plan(75, 56, 148, 0)[74] == [(74, 0, 56, 74, 74)]  # not two workers for every tile


def test_workspace_bytes(sp):
    assert sp.linear_workspace_bytes(1, 9216, 16, 9216, True) > 0
    assert sp.linear_workspace_bytes(64, 2048, 96, 4096, False) > 0
    for bad in [(0, 128, 16, 128, True), (1025, 128, 16, 128, True), (1, 0, 16, 128, True), (1, 128, -1, 128, True), (1, 128, 16, 0, True),
                (1, 128, 16, 24, True), (1, 128, 16, 12, False)]:
        assert sp.linear_workspace_bytes(*bad) == 0, bad


def test_c_boundary_refuses_before_any_cuda_call(sp):
    lib, p, odd = sp.spmm_api.LIB, ctypes.c_void_p(4096), ctypes.c_void_p(4100)
    quant = lib.spmm_b200_quantize_fp8
    assert quant(None, p, 0, 1, 0, 128, 1, p, p) == 0  # nothing to do
    for args in [(p, 2, 1, 4, 128, 1, p, p), (p, 0, 0, 4, 128, 1, p, p), (p, 0, 2, 4, 128, 1, p, p), (p, 0, 1, -1, 128, 1, p, p),
                 (p, 0, 1, 4, 120, 1, p, p), (p, 0, 1, 4, 0, 1, p, p), (p, 0, 1, 4, 128, 64, p, p), (None, 0, 1, 4, 128, 1, p, p),
                 (p, 0, 1, 4, 128, 1, None, p), (p, 0, 1, 4, 128, 1, p, None), (odd, 0, 1, 4, 128, 1, p, p), (p, 0, 1, 4, 128, 1, odd, p)]:
        assert quant(None, *args) == 1, args
    fp8 = lib.spmm_b200_fp8_linear
    assert fp8(None, None, None, None, None, None, 0, 128, 0, 128, None, 0) == 0
    good = [p, p, p, p, p, 0, 128, 16, 128, None, 0]
    for at, value in [(0, None), (1, None), (2, None), (3, None), (4, None), (0, odd), (2, odd), (5, 2), (5, -1), (6, 0), (7, -1), (8, 0),
                      (8, 120), (9, odd), (4, ctypes.c_void_p(4097))]:
        args = list(good)
        args[at] = value
        assert fp8(None, *args) == 1, (at, value)
    grouped = lib.spmm_b200_grouped_linear
    good = [p, p, p, 1, p, 4, 128, 16, 128, None, 0]
    for at, value in [(0, None), (1, None), (2, None), (3, 2), (4, None), (4, ctypes.c_void_p(4098)), (5, 0), (5, 1025), (6, 0), (7, -1),
                      (8, 0), (8, 12), (0, odd), (1, odd)]:
        args = list(good)
        args[at] = value
        assert grouped(None, *args) == 1, (at, value)
    grouped8 = lib.spmm_b200_grouped_fp8_linear
    good = [p, p, p, p, p, 0, p, 4, 128, 16, 128, None, 0]
    for at, value in [(0, None), (1, None), (3, None), (4, None), (6, None), (5, 3), (7, 0), (8, -128), (10, 24)]:
        args = list(good)
        args[at] = value
        assert grouped8(None, *args) == 1, (at, value)


def test_sizes_that_indices_cannot_hold_are_refused(sp):
    """The last tile's columns have to have numbers that fit an int, and a row of K byte offsets that do; a 16-bit depth is
    one accumulation, which has to end before a wait gives up."""
    lib, p = sp.spmm_api.LIB, ctypes.c_void_p(4096)
    most = 2 ** 31 - 513
    for n in (most + 1, 2 ** 31 - 256, 2 ** 31 - 1):
        assert sp.linear_workspace_bytes(1, 128, n, 16, True) == 0
        assert sp.linear_workspace_bytes(3, 128, n, 16, False) == 0
        assert lib.spmm_b200_fp8_linear(None, p, p, p, p, p, 0, 128, n, 16, None, 0) == 1
        assert lib.spmm_b200_grouped_linear(None, p, p, p, 0, p, 3, 128, n, 16, None, 0) == 1
        assert lib.spmm_b200_grouped_fp8_linear(None, p, p, p, p, p, 0, p, 3, 128, n, 16, None, 0) == 1
    for n, k, eight, fits in [(most, 16, True, True), (most, 16, False, True), (16, 2 ** 29, True, True), (16, 2 ** 29 + 16, True, False),
                              (16, 2 ** 27, False, True), (16, 2 ** 27 + 8, False, False)]:
        assert (sp.linear_workspace_bytes(1, 128, n, k, eight) > 0) == fits, (n, k, eight)
    assert lib.spmm_b200_grouped_linear(None, p, p, p, 0, p, 3, 128, 16, 2 ** 27 + 8, None, 0) == 1


def test_python_sizes_longer_than_an_int_are_refused(sp):
    """2^32 + 128 would arrive at the C boundary as 128."""
    import torch
    far = 2 ** 32 + 128
    for at in range(4):
        sizes = [1, 128, 16, 128]
        assert sp.linear_workspace_bytes(*sizes, True) > 0
        sizes[at] = far
        assert sp.linear_workspace_bytes(*sizes, True) == 0
        t = torch.zeros((16, 128), dtype=torch.bfloat16)
        if at > 0:
            with pytest.raises(ValueError, match="sizes"):
                sp.fp8_linear(None, t, t, t, t, t, *sizes[1:], None)
        with pytest.raises(ValueError, match="sizes"):
            sp.grouped_linear(None, t, t, t, t, *sizes, None)
        with pytest.raises(ValueError, match="sizes"):
            sp.grouped_fp8_linear(None, t, t, t, t, t, t, *sizes, None)
    with pytest.raises(ValueError, match="sizes"):
        sp.quantize_fp8(None, torch.zeros((far, 0, 16), dtype=torch.bfloat16), t, t, 128)
    with pytest.raises(ValueError, match="sizes"):
        sp.fp8_linear(None, t, t, t, t, t, 128, -1, 128, None)


def test_wait_selftest_refuses_limits_out_of_range(sp):
    for limit_ms in (0, 1001, 2 ** 32 - 1):
        assert sp.spmm_api.LIB.spmm_b200_selftest_linear_wait_timeout(None, limit_ms) == 1
