"""The paged store where its arithmetic and its shared state can go wrong: zeros,
infinities and values of unlike size beside one another, extreme windows, streams and
workspaces.  Cases, the 64-bit reference and its tolerances are test_pages.py's."""
import math

import pytest

from test_pages import Case, env  # noqa: F401  (env is a fixture)

pytestmark = pytest.mark.gpu


def rewrite(c, k=None, v=None):
    """The whole sequences again with other keys or values."""
    c.k = c.k if k is None else k.to(c.dtype)
    c.v = c.v if v is None else v.to(c.dtype)
    c.store.write_dev(c.whole, c.k, c.v)


# ------------------------------------------------------------------ zeros


@pytest.mark.parametrize("bits,kind", [(16, "bf16"), (8, "bf16"), (8, "f16"), (4, "bf16")])
@pytest.mark.parametrize("q,k", [(0.0, 1.0), (1.0, 0.0), (0.0, 0.0), (0.0, 1e-3), (1e-3, 0.0)])
@pytest.mark.parametrize("new", [1, 70])
def test_zero_queries_and_keys(env, bits, kind, q, k, new):
    """Scores of zero are equal weights for what a row sees."""
    c = Case(env, [new], [200], heads=1, bits=bits, kind=kind)
    rewrite(c, k=c.k * k)
    c.check(c.queries() * q, 0.1)
    c.check(c.queries() * q, 0.1, 33, 5)


@pytest.mark.parametrize("bits", [16, 8, 4])
@pytest.mark.parametrize("size", [0.25, 1e-4])
def test_scale_zero(env, bits, size):
    c = Case(env, [70], [200], heads=1, bits=bits)
    rewrite(c, k=c.k * size)
    c.check(c.queries() * size, 0.0)
