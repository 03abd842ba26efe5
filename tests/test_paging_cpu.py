"""CPU: the index arithmetic of the paged cache and of the attention's work split
(ocelotl_b200/csrc/paging.cuh, the same source the kernels are built from)."""
import ctypes as C
import subprocess
from pathlib import Path

import numpy as np
import pytest

HERE = Path(__file__).resolve().parent
TILE = 64


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    so = tmp_path_factory.mktemp("paging") / "paging.so"
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", str(HERE / "paging_host.cpp"), "-o", str(so)], check=True)
    lib = C.CDLL(str(so))
    lib.walk.restype = C.c_longlong
    lib.walk.argtypes = [C.c_void_p, C.c_void_p, C.c_longlong, C.c_int, C.c_int, C.c_int, C.c_uint, C.c_uint, C.c_int, C.c_int, C.c_void_p, C.c_longlong]
    lib.place.argtypes = [C.c_void_p] + [C.c_longlong] * 3 + [C.c_uint, C.c_longlong, C.c_int, C.c_void_p, C.c_void_p]
    lib.wrong_quotient.restype = C.c_longlong
    lib.wrong_quotient.argtypes = [C.c_uint] + [C.c_longlong] * 3
    return lib


def walk(lib, positions, cap, items, ctas, snap=0, min_share=1, seqs=None, n_seqs=None, together=1):
    pos = np.asarray(positions, np.int32)
    sq = None if seqs is None else np.asarray(seqs, np.int32)
    room = int(sum(-(-(min(p + 1, cap)) // TILE) for p in pos.astype(int) if p >= 0)) * items + 1
    out = np.full((room, 4), -1, np.int32)
    n = lib.walk(pos.ctypes.data, None if sq is None else sq.ctypes.data, len(pos) if n_seqs is None else n_seqs, len(pos),
                 cap, items, ctas, min_share, snap, together, out.ctypes.data, room)
    assert n >= 0, n
    return out[:n]


@pytest.mark.parametrize("positions,items,ctas", [
    ([0], 1, 296), ([554], 8, 296), ([130999], 8, 296), ([130999], 1, 444), ([-1, -1], 8, 296), ([63, 64, 65, -1, 127], 3, 7),
    ([5] * 230, 2, 444), (list(range(0, 4000, 37)), 16, 296), ([-1, 700, -1, -1, 3, -1], 1, 5), ([2147483647], 2, 148),
    ([100000, 0, 0, 0, 0], 8, 148),
])
def test_every_tile_once_and_shares_agree(lib, positions, items, ctas):
    cap = 140000
    for snap in (1, 2, 5, 64):
        moved = walk(lib, positions, cap, items, ctas, snap, min_share=1 + snap % 4)
    got = walk(lib, positions, cap, items, ctas)
    assert np.array_equal(moved[:, :3], got[:, :3])
    want = [(r, i, t) for r, p in enumerate(positions) if p >= 0
            for i in range(items) for t in range(-(-min(p + 1, cap) // TILE))]
    assert [tuple(x[:3]) for x in got.tolist()] == want
    if len(want):
        # without moved cuts every run has an equal share of units (a tile, or an item's start), but for one
        # unit of rounding and the one that a cut within an item's start moves at either end
        total = len(want) + sum(1 for p in positions if p >= 0) * items
        cost = np.bincount(got[:, 3]) + np.bincount(got[got[:, 2] == 0][:, 3], minlength=got[:, 3].max() + 1)
        assert cost.max() <= -(-total // min(ctas, total)) + 2


def test_random_batches(lib):
    rng = np.random.default_rng(3)
    for _ in range(200):
        rows = int(rng.integers(1, 40))
        pos = np.where(rng.random(rows) < 0.2, -1, rng.integers(0, int(rng.choice([2, 70, 900, 9000])), rows))
        walk(lib, pos, int(rng.integers(1, 9000)), int(rng.integers(1, 17)), int(rng.integers(1, 300)),
             snap=int(rng.integers(0, 9)), min_share=int(rng.integers(1, 12)))


def test_short_items_are_not_shared(lib):
    got = walk(lib, [255] * 16, 4096, 8, 296, snap=2)  # 128 items of 4 tiles
    owners = {}
    for r, i, _, c in got.tolist():
        owners.setdefault((r, i), set()).add(c)
    assert all(len(v) == 1 for v in owners.values())


def test_rows_of_unknown_sequences_have_no_tiles(lib):
    got = walk(lib, [100, 100, 100, 100], 1000, 2, 10, seqs=[0, -1, 2, 1], n_seqs=2)
    assert sorted(set(got[:, 0].tolist())) == [0, 3]


@pytest.mark.parametrize("together", [2, 4, 8])
def test_rows_of_a_sequence_share_items(lib, together):
    rng = np.random.default_rng(together)
    for _ in range(100):
        rows, n_seqs, items = int(rng.integers(1, 50)), int(rng.integers(1, 6)), int(rng.integers(1, 5))
        seqs = np.repeat(rng.integers(-1, n_seqs + 1, rows), rng.integers(1, 12, rows))[:rows]  # -1 and n_seqs are unknown
        pos = np.where(rng.random(rows) < 0.2, -1, rng.integers(0, int(rng.choice([2, 70, 900, 9000])), rows))
        cap = int(rng.integers(1, 9000))
        got = walk(lib, pos, cap, items, int(rng.integers(1, 300)), int(rng.integers(0, 4)), int(rng.integers(1, 4)), seqs, n_seqs, together)
        want, r = [], 0
        while r < rows:
            n = 1
            while r + n < rows and (r + n) % together and seqs[r + n] == seqs[r]:
                n += 1
            tokens = max(min(int(p) + 1, cap) for p in pos[r:r + n]) if 0 <= seqs[r] < n_seqs else 0
            want += [(r, i, t) for i in range(items) for t in range(-(-tokens // TILE))]
            r += n
        assert [tuple(x[:3]) for x in got.tolist()] == want


def test_place_of(lib):
    table = np.array([[3, 7, -1, 99], [5, 9, 0, 1]], np.int32)
    page, slot = C.c_int(-5), C.c_int(-5)

    def place(seq, tok, n_pages=10, max_pages=4, size=24):
        ok = lib.place(table.ctypes.data, max_pages, 4, n_pages, size, seq, tok, C.byref(page), C.byref(slot))
        return (page.value, slot.value) if ok else None

    assert place(0, 0) == (3, 0) and place(0, 23) == (3, 23) and place(0, 24) == (7, 0) and place(1, 95) == (1, 23)
    assert place(0, 48) is None      # page -1
    assert place(0, 72) is None      # page past the cache
    assert place(1, 96) is None      # past the table
    assert place(1, 48, max_pages=2) is None
    assert place(1, 2147483647) is None
    assert place(1, 2, size=1) == (0, 0)


def test_quotients(lib):
    top = 2**31
    divisors = list(range(1, 200)) + [255, 256, 257, 1000, 4095, 4096, 4097, 65535, 65536, 10**6, 2**30 - 1, 2**30, 2**30 + 1,
                                      2**31 - 1]
    for d in divisors:
        assert lib.wrong_quotient(d, 0, 70000, 1) == -1
        assert lib.wrong_quotient(d, top - 70000, top, 1) == -1
        assert lib.wrong_quotient(d, 0, top, 10007) == -1
        first = (top // d) * d  # around the last multiple
        assert lib.wrong_quotient(d, max(0, first - 5), min(top, first + 5), 1) == -1
