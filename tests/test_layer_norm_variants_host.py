"""The compiled variants of the layer norm kernels are those that some call reaches, and no others: the rule of the launches,
restated here over every number of columns, against the kernel names in the built library."""
import re

from elixir_amd import _ops_abi

DTYPES = {0: 4, 1: 2, 2: 2}    # code of the type: bytes
MAX_COLS = 16384


def up(n):
    """The next power of two."""
    return 1 << (n - 1).bit_length()


def by_rows(rows, cols, v):
    """(accesses per lane, wavefronts per row, lanes per row)"""
    accesses = -(-cols // (64 * v))
    if accesses >= (17 if v == 1 else 8) or (rows < 4096 and accesses >= 4):
        return up(-(-accesses // 4)), 4, 64
    for lanes in (4, 8, 16, 32):
        if cols <= lanes * v:
            return 1, 1, lanes
    return up(accesses), 1, 64


def backward(rows, cols, v, size):
    """(accesses, wavefronts, lanes, streams past the cache)"""
    stream = int(v > 1 and 2 * rows * cols * size > 256 << 20)
    for lanes in (4, 8, 16, 32):
        if cols <= lanes * v:
            return 1, 1, lanes, stream
    waves = 1
    while waves < 16 and waves * 512 < cols:
        waves *= 2
    return up(-(-cols // (waves * 64 * v))), waves, 64, stream


def test_every_compiled_variant_has_a_caller():
    want = {'fwd': set(), 'few': set(), 'bwd': set()}
    for d, size in DTYPES.items():
        for v in (1, 16 // size):
            for cols in range(v, MAX_COLS + 1, v):
                want['few'].add((d, v) + by_rows(1024, cols, v))
                want['fwd'].update((d, v) + by_rows(rows, cols, v) for rows in (1, 4095, 4096))
                want['bwd'].update((d, v) + backward(rows, cols, v, size) for rows in (1025, 1 << 30))
    with open(_ops_abi.LIB_PATH, 'rb') as f:
        names = set(re.findall(rb'layer_norm_(fwd|few|bwd)_kernelI((?:L[ib]\d+E)+)', f.read()))
    built = {kind: set() for kind in want}
    for kind, args in names:
        built[kind.decode()].add(tuple(int(x) for x in re.findall(rb'L[ib](\d+)E', args)))
    for kind in want:
        assert built[kind] == want[kind], (kind, 'no caller', sorted(built[kind] - want[kind]), 'missing', sorted(want[kind] - built[kind]))
