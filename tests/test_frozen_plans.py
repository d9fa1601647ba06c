"""Host side: every way a product of the 8-bit frozen layer and of the gated projection can be run is run by a GPU test (no GPU needed: the rule is
the library's, lyc_frozen_plan)."""
import math
import random

from frozen_plans import BASE, INT8, KEEP, PLANS, PRODUCTS
from lycoris_amd import _native as N


def plan(product, M, K, n, dtype, flags):
    v = N.load().lyc_frozen_plan(product, M, K, n, dtype, flags)
    assert v > 0
    return v & 0xffff, int(v >> 16 > 1)


def kind(product, dtype, flags, tile, parts):
    return product, dtype, product < 2 or bool(flags & INT8), tile, parts


def test_the_table_is_what_the_library_does():
    for product, dtype, M, K, n, flags, tile, parts in PLANS:
        assert plan(product, M, K, n, dtype, flags) == (tile, parts), (PRODUCTS[product], dtype, M, K, n, flags)


def test_nothing_is_chosen_that_the_table_has_not():
    tested = {kind(p, dt, flags, tile, parts) for p, dt, _, _, _, flags, tile, parts in PLANS}
    rng = random.Random(5)
    spread = lambda hi: int(round(math.exp(rng.uniform(0.0, math.log(hi)))))  # noqa: E731
    for _ in range(60000):
        product, dtype = rng.randrange(5), rng.randrange(3)
        flags = rng.choice([0, INT8]) * (product in (2, 3)) | (rng.choice([0, KEEP]) | rng.choice([0, BASE])) * (product == 2)
        M, K, n = spread(40000), spread(16000), spread(16000)
        assert kind(product, dtype, flags, *plan(product, M, K, n, dtype, flags)) in tested, (PRODUCTS[product], dtype, M, K, n, flags)


def test_bad_arguments():
    lib = N.load()
    assert [lib.lyc_frozen_plan(*a) for a in ((5, 4, 4, 4, 0, 0), (-1, 4, 4, 4, 0, 0), (0, 4, 0, 4, 0, 0), (0, 4, 4, 4, 3, 0), (2, 4, 4, 0, 2, 0))] == [-1] * 5
