"""Where what is not finite goes in the gated delta rule: a value stays in its column, a key, decay or rate in its head, a query in its row; and from its
token on every result there is not finite either, by both forms, in both types, whatever number of heads share the key."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

from test_gpu_delta import delta_case
from test_gpu_ssm import GUARD

DV = 32
SHAPES = [(4, 4, 32), (4, 2, 128), (2, 1, 200)]  # heads, heads of keys, key_dim


def spoilt_case(name, value, shape, dtype, form, grows=False, **kw):
    heads, kh, dk = shape
    n, at, one = {"one": (1, 0, True), "tokens": (9, 4, False), "chunks": (150, 40, False), "second chunk": (150, 64, False)}[form]
    share = heads // kh
    head = heads - 1  # of a value, a decay, a rate or a state; a key's and a query's is that of `mine`
    mine = head // share

    def spoil(x, rates, biases, S):
        row = at + (0 if one else GUARD)
        if name == "v":
            x[2][row, head * DV + 3] = value
        elif name == "k":
            x[1][row, mine * dk + 7] = value
        elif name == "q":
            x[0][row, mine * dk + 5] = value
        elif name == "beta":
            x[4][row, head] = value
        elif name == "dt":
            x[3][row, head] = value
        else:
            S[0, head, 4, 3] = value

    def look(y, left, starts, x, S0):
        return y[starts[0]:starts[1], :heads * DV].reshape(n, heads, DV).astype(np.float32), left[0]
    run = dict(dtype=dtype, one=one, check=look, **kw)
    clean, want = delta_case(heads, kh, dk, DV, [n], **run)
    y, S = delta_case(heads, kh, dk, DV, [n], change=spoil, **run)
    ybad, Sbad = np.zeros(y.shape, bool), np.zeros(S.shape, bool)
    heads_of_key = slice(mine * share, (mine + 1) * share)
    if name == "v":
        ybad[at:, head, 3] = Sbad[head, :, 3] = True
    elif name == "state":
        ybad[:, head, 3] = Sbad[head, :, 3] = True
    elif name == "q":
        ybad[at, heads_of_key] = True
    elif name == "k":
        ybad[at:, heads_of_key] = Sbad[heads_of_key] = True
    else:
        ybad[at:, head] = Sbad[head] = True
    ahead = np.zeros(y.shape, bool)
    if grows:  # 64 rows share powers of two that the largest decay sets: of rows ahead in this head either run is within the roundings of its 2 x 64 products
        ahead[:at, head] = True
        with np.errstate(invalid="ignore"):
            off, size = np.abs(y - clean), np.abs(clean).max(2, keepdims=True)
            assert (off <= size * (2.0 ** -14 if dtype == "f32" else 2.0 ** -10))[ahead].all()
    same = ~ybad & ~ahead
    assert np.array_equal(y[same], clean[same]) and np.array_equal(S[~Sbad], want[~Sbad])  # (of binary16 some that grew are infinite in both)
    assert not np.isfinite(y[ybad]).any() and not np.isfinite(S[Sbad]).any()


@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("name", ["v", "k", "q", "state"])
@pytest.mark.parametrize("form", ["one", "tokens", "chunks", "second chunk"])
@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("shape", SHAPES)
def test_values_keys_queries_and_states(shape, dtype, form, name, value):
    spoilt_case(name, value, shape, dtype, form)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("form", ["one", "tokens", "chunks"])
@pytest.mark.parametrize("shape", SHAPES)
def test_rates(shape, form, dtype):
    spoilt_case("beta", np.nan, shape, dtype, form)
    for value in (np.nan, np.inf, -np.inf):
        spoilt_case("beta", value, shape, dtype, form, sigmoid=0)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("form", ["one", "tokens", "chunks"])
@pytest.mark.parametrize("shape", SHAPES)
def test_decays_that_are_no_number(shape, form, dtype):
    spoilt_case("dt", np.nan, shape, dtype, form)


@pytest.mark.parametrize("softplus", [1, 0])
@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("form", ["one", "tokens", "chunks"])
@pytest.mark.parametrize("shape", SHAPES)
def test_decays_that_grow_without_end(shape, form, dtype, softplus):
    """The logarithm is plus infinity: not a number that some clip makes finite"""
    spoilt_case("dt", np.inf, shape, dtype, form, grows=True, softplus=softplus, A=False)
