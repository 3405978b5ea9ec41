"""Sizes at which index arithmetic of the 4-bit attention and of the step tables would
leave its range are refused (no GPU needed)."""
import pytest

from test_fp4_cpu import ALIGN, P16, UNSUPPORTED, _decode, _tables

WIDE = dict(batch=1, hq=1, hkv=1, q=P16 + 2)   # what is not refused goes on to the alignment


def _reciprocal(tpp):
    return -(-(1 << 32) // tpp)


def _exact(tpp, tiles):
    """The page of every tile below `tiles` follows from the reciprocal: the last tile of a page
    is the first to go wrong, and the later the page the sooner."""
    last = tiles // tpp * tpp - 1
    return all((x * _reciprocal(tpp)) >> 32 == x // tpp
               for x in (last, last - tpp, tiles - 1) if x >= 0)


@pytest.mark.parametrize("page", [48, 80, 112, 144, 1008, 4112, 16400, 65552, 100016, 1000016])
def test_page_numbers_are_exact_or_refused(page):
    tpp = page // 16
    most = ((1 << 31) - 1) // page
    lo, hi = 1, most + 1        # lo pages a row are accepted, hi are not
    assert _decode(page=page, maxp=lo, pt_sb=lo, **WIDE) == ALIGN
    while hi - lo > 1:
        mid = (lo + hi) // 2
        rc = _decode(page=page, maxp=mid, pt_sb=mid, **WIDE)
        assert rc in (ALIGN, UNSUPPORTED)
        lo, hi = (mid, hi) if rc == ALIGN else (lo, mid)
    assert _exact(tpp, lo * tpp)
    for pages in range(max(1, lo - 300), lo + 1):
        assert _exact(tpp, pages * tpp)
    # hardly anything is refused without need: most sizes up to 2^31 tokens, and the pages
    # beyond an earlier limit are wrong ones
    if lo < most:
        over = _reciprocal(tpp) * tpp - (1 << 32)
        assert (lo + 1) * tpp * over > 1 << 32


def test_wrong_page_numbers_exist():
    """What the limits are for: a sequence of 1.8 10^7 tokens in pages of 65,552."""
    x = 274 * 4097 - 1
    assert (x * _reciprocal(4097)) >> 32 != x // 4097
    assert _decode(page=65552, maxp=274, pt_sb=274, **WIDE) == UNSUPPORTED
    assert _decode(page=65552, maxp=250, pt_sb=250, **WIDE) == ALIGN


def test_step_tables_whose_loops_would_pass_32_bits():
    """Threads step through rows and pages in strides of 16 * 1024 * 4."""
    most = 2 ** 31 - 2 ** 17
    for n in (2 ** 31 - 1, 2 ** 31 - 65536, most + 1):
        assert _tables(n=n) == UNSUPPORTED
    wide = most // 4096
    assert _tables(batch=4096, maxp=wide + 1, sb=wide + 1, page=16) == UNSUPPORTED
