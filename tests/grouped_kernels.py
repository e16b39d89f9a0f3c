"""Which kernel a product by expert runs, restated on the host from the rule in csrc/grouped_tile.hip (``choose``, ``whole_rows``): what a
test of a kernel needs in order to know that its sizes reach it."""


def _tiles(S, groups, cols, bm, bn):
    t = S // bm + groups // 2 if groups > 1 else -(-S // bm)
    return max(t, groups) * -(-cols // bn)


def _kind(rows, b_rows, aligned, whole, S, E, K, N, each, element, grouped):
    """K: length of a row of the left operand (rows), else its columns; N: columns of the result."""
    groups = min(S, E) if grouped else 1
    size = (S, groups, N) if rows else (K, 1, N)
    large = max(1250, 1460 * each * _tiles(*size, 256, 256) // 256)
    small = max(600, 480 * each * _tiles(*size, 128, 128) // 256)
    any_ = max(1150, 1200 * each * _tiles(*size, 128, 128) // 256)
    tile = any_ if not aligned else min(large, small)
    if rows:
        n1, n2 = (_tiles(*size, bm, 16 if b_rows else 128) for bm in (16, 32))
        few1 = max(82, 105 * n1 // 256) if b_rows else 282 * -(-n1 // 256)
        few2 = max(100, 154 * n2 // 256) if b_rows else 358 * -(-n2 // 256)
        if min(few1, few2) < tile and K * element >= 16 and N >= 8 and S < 1 << 19:
            return "few1" if few1 <= few2 else "few2"
    if not aligned:
        return "any"
    return ("large" if large < small else "small") + ("" if whole else "_cut")


def _at(numbers, n):
    return all(v % n == 0 for v in numbers)


def forward(S, E, K, N, moved=0):
    """Products of 16-bit rows; `moved`: bytes by which the operands begin behind an aligned address."""
    return _kind(True, False, _at((2 * K, 2 * N, moved), 4), _at((2 * K, 2 * N, moved), 16), S, E, K, N, 1, 2, True)


def rows_gradient(S, E, K, N, moved=0):
    return _kind(True, True, _at((2 * N, moved), 4), _at((2 * N, 2 * K, moved), 16), S, E, N, K, 1, 2, True)


def weights_gradient(S, E, K, N, moved=0, element=2):
    at = (2 * K, 2 * N, moved)
    return _kind(False, False, _at(at, 4), _at((*at, element * N), 16), S, E, K, N, E, 2, True)


def int8(S, E, K, N, moved=0, element=2, grouped=True):
    return _kind(True, True, _at((K, moved), 4), _at((K, moved, element * N), 16), S, E, K, N, 1, 1, grouped)
