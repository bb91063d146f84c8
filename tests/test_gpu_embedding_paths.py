"""The embedding gradient, exactly, on every path of its kernels. Gradients are -1, 0 and 1, sums of which float32 holds
exactly in any order: a token that is lost, doubled or added to another row shows, however long its run is."""

import math

import pytest
import torch

DEV = "cuda"
DTYPES = [torch.float32, torch.bfloat16, torch.float16]  # in the order of fc_dtype

# name: (n, rows, width, kind of ids, path)
CASES = {
    # sorted by one workgroup: up to 1,024 and 4,096 tokens, one to four passes of 8 bits
    "one workgroup, 1 key each": (900, 200, 40, "uniform", "block"),
    "one workgroup, 3 passes": (4096, 120000, 29, "zipf", "block"),
    "one workgroup, 4 passes": (1025, (1 << 24) + 5, 1, "uniform", "block"),
    # tiles of 1,024 keys
    "tiles of 1,024": (65536, 5000, 24, "uniform", "tiles4"),
    "tiles of 1,024, 4 passes": (5000, (1 << 24) + 5, 2, "ends", "tiles4"),
    # tiles of 2,048, counts added in the placement
    "tiles of 2,048": (70000, 5000, 24, "uniform", "tiles8"),
    # counts summed by a launch of their own; more runs to join than workgroups, short ones
    "scanned, batches of short joins": (300000, 120000, 29, "uniform", "scan"),
    # short and long runs in one batch
    "scanned, runs of all lengths": (300000, 120000, 29, "zipf", "scan"),
    "scanned, 1 pass": (300001, 129, 48, "zipf", "scan"),
    # one run of 18,751 pieces, and a few others
    "scanned, one run": (300005, 120000, 3, "same", "scan"),
    # long pieces, rows of several workgroups in the joins
    "long pieces": (70000, 3000, 1030, "zipf", "tiles8"),
    # sums per wave, nothing sorted
    "few rows": (300001, 4, 16, "uniform", "few"),
    "few rows, one": (70001, 1, 1, "uniform", "few"),
    "few rows, odd": (20011, 31, 100, "zipf", "few"),
    "few rows, wide": (2500, 7, 1030, "uniform", "few"),
}


def _ids(n, rows, kind):
    gen = torch.Generator().manual_seed(n + rows)
    u = torch.rand(n, generator=gen, dtype=torch.float64)
    if kind == "same":
        ids = torch.full((n,), rows // 2, dtype=torch.int64)
        ids[::40001] = torch.arange(ids[::40001].numel())
    elif kind == "ends":
        ids = torch.where(u < 0.5, (u * 200).long(), rows - 1 - ((1 - u) * 200).long())
    else:
        ids = (u * rows if kind == "uniform" else torch.exp(u * math.log(rows + 1)) - 1).long()
    ids.clamp_(0, rows - 1)
    outside = torch.tensor([-1, rows, 1 << 40, -(1 << 62)])
    ids[3::97] = outside[torch.arange(ids[3::97].numel()) % 4]
    return ids


def _plan(case, dtype):
    """(path, tokens of a piece): the plan whose workspace has the size that the library asks for, of all that there are."""
    from flashcart_amd import _lib
    n, rows, width, _, _ = CASES[case]
    size = torch.empty((), dtype=dtype).element_size()
    chunk = 16 // size
    need = _lib.load().fc_embedding_bwd_workspace(DTYPES.index(dtype), n, rows, width)
    up = lambda b: -(-b // 256) * 256  # noqa: E731

    def sorted_bytes(tile, length):
        tiles, pieces = -(-n // tile), -(-n // length)
        return 4 * up(4 * n) + up(1024 * tiles) + 1024 + 2 * up(4 * pieces * width) + up(4 * pieces) + 256

    sizes = {(tile, 1 << k): sorted_bytes(tile, 1 << k) for tile in (1024, 2048) for k in range(4, 11)}
    found = [key for key, b in sizes.items() if b == need]
    if not found:
        assert need % (4 * rows * -(-width // chunk) * chunk) == 0
        return "few", 0
    assert len({length for _, length in found}) == 1
    if n <= 4096:
        return "block", found[0][1]
    assert len(found) == 1
    tile, length = found[0]
    return "tiles4" if tile == 1024 else "tiles8" if -(-n // tile) <= 64 else "scan", length


def _runs(ids, rows, padding, length):
    """Pieces of each run that more than one piece holds."""
    dead = (ids < 0) | (ids >= rows) | (ids == padding)
    keys = torch.where(dead, rows, ids).sort().values
    cut = torch.arange(length, keys.numel(), length)
    crossing = keys[cut][(keys[cut] == keys[cut - 1]) & (keys[cut] < rows)]
    return crossing.unique(return_counts=True)[1] + 1


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", CASES)
def test_cases_take_their_path(case, dtype):
    """(no GPU needed) A changed threshold does not move a case to another path unnoticed."""
    n, rows, width, kind, path = CASES[case]
    got, length = _plan(case, dtype)
    assert got == path
    if path == "few":
        return
    assert (length > 16) == (case == "long pieces")
    runs = _runs(_ids(n, rows, kind), rows, _padding(rows), length)
    joins, short = runs.numel(), int((runs <= 4).sum())
    if "batches" in case:
        assert joins > 4096 and short == joins
    if "all lengths" in case:
        assert joins > 4096 and 0 < short < joins and int(runs.max()) > 256
    if "one run" in case:
        assert joins == 1 and int(runs.max()) > 65536 // 4


def _padding(rows):
    return rows // 3 if rows > 1 else -1


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", CASES)
def test_gradient_is_exact(case, dtype):
    n, rows, width, kind, _ = CASES[case]
    print(f"embedding gradient {case}: n={n} rows={rows} width={width} {kind} {dtype}", flush=True)
    ids, padding = _ids(n, rows, kind), _padding(rows)
    live = (ids >= 0) & (ids < rows) & (ids != padding)
    gen = torch.Generator(device=DEV).manual_seed(width)
    grad = torch.randint(-1, 2, (n, width), device=DEV, generator=gen).to(dtype)
    ids, live = ids.to(DEV), live.to(DEV)
    # (float64 sums of integers: exact too; rounded once, as the kernels' float32 sums are)
    want = torch.zeros(rows, width, dtype=torch.float64, device=DEV).index_add_(0, ids[live], grad[live].double())
    grad[~live] = math.nan  # adds to no row
    got = torch.ops.flashcart.embedding_bwd(grad, ids, rows, 1.0, padding)
    wrong = got != want.float().to(dtype)
    assert not wrong.any(), f"{int(wrong.sum())} elements of {int(wrong.any(1).sum())} rows"
