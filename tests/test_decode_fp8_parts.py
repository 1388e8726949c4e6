"""What the kernel that joins the parts of an 8-bit decode takes as indices, when a wait of the kernel in front of it has run out and
the workspace holds whatever it held: none outside the workspace, and none refused that a finished kernel leaves. No GPU."""
import random

import pytest

import hipkittens_b200 as hk
from hipkittens_b200 import _native

ENDS = (-2 ** 31, -2 ** 31 + 1, -1000, -1, 0, 1, 2, 2 ** 30, 2 ** 31 - 2, 2 ** 31 - 1)


def parts_of(first, group, last, hkv, kvh):
    return [first] + [2 * ((group + i) * hkv + kvh) for i in range(1, last - group + 1)]


@pytest.mark.parametrize("groups,hkv,d", [(2368, 1, 128), (296, 8, 64), (182, 13, 128), (1, 65535, 64), (1, 1, 64)])
def test_whatever_is_followed_lies_in_the_workspace(native_built, groups, hkv, d):
    follows = hk.capi().hk_selftest_decode_fp8_parts
    n_parts = 2 * groups * hkv
    assert n_parts * 8 * (d + 2) * 4 <= hk.paged_decode_fp8_workspace_bytes(1, hkv, d)
    rng = random.Random(groups)
    near = [x + e for x in (0, groups, n_parts, groups // 2) for e in (-1, 0, 1)]
    tries = [(f, g, l) for f in (*ENDS, *near) for g in (*ENDS, *near) for l in (*ENDS, *near)]
    tries += [tuple(rng.randint(-2 ** 31, 2 ** 31 - 1) for _ in range(3)) for _ in range(2000)]
    tries += [(rng.randint(-5, n_parts + 5), rng.randint(-5, groups + 5), rng.randint(-5, groups + 5)) for _ in range(2000)]
    taken = 0
    for first, group, last in tries:
        if follows(first, group, last, groups, hkv):
            taken += 1
            assert last - group < groups
            assert all(0 <= x < n_parts for kvh in (0, hkv - 1) for x in parts_of(first, group, last, hkv, kvh))
    assert taken


def test_what_a_finished_kernel_leaves_is_followed(native_built):
    """The kernel's arithmetic: group w of n has the places [T w / n, T (w + 1) / n) of the row of all pages."""
    follows = hk.capi().hk_selftest_decode_fp8_parts
    rng = random.Random(1)
    for _ in range(200):
        hkv, pages = rng.choice([1, 2, 5, 8, 13, 400]), [rng.randint(0, rng.choice([3, 40, 3000])) for _ in range(rng.randint(1, 70))]
        row_groups, total = max(2368 // hkv, 1), sum(pages)
        n = min(row_groups, -(-total // 8))
        begin = 0
        for count in pages:
            if count:
                group, last = (((at + 1) * n - 1) // total for at in (begin, begin + count - 1))
                assert total * group // n <= begin < total * (group + 1) // n
                for head in (0, hkv - 1):
                    warp = group * hkv + head
                    assert all(follows(first, group, last, row_groups, hkv) == 1 for first in (2 * warp, 2 * warp + 1))
            begin += count


def test_refusals(native_built):
    follows = hk.capi().hk_selftest_decode_fp8_parts
    assert follows(0, 0, 0, 0, 8) == follows(0, 0, 0, 5, 0) == follows(0, 0, 0, 2 ** 20, 65535) == _native.HK_EINVAL
