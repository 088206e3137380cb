"""Normed and rotated heads, 4-bit cache, decay attention: numbers of very different sizes side by side.  Every row is held to its own size.

Tolerances.  A bf16 result is rounded by half a step, 2^-8 of it at most; fp16 operands by 2^-12 of themselves (standard deviation 2^-12 / sqrt(3)), at random."""
import numpy as np
import pytest

from oracle import layer_stack as O
from rotated_helpers import Decay, Quantized, f64, stream, tables
from test_gpu_rotated_mixers import CHUNK, FLASH, SCAN, SIMT, STREAM, cfg4, cfgd

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _built(cuda, stack_lib):
    stack_lib.tbl_device_status(stream(cuda))
    yield
    assert stack_lib.tbl_device_status(stream(cuda)) == 0


def own_rows_close(got, want, tol, what):
    err = np.sqrt(((got - want) ** 2).mean(axis=1)) / np.sqrt((want ** 2).mean(axis=1))
    worst = int((err / tol).argmax())
    assert np.isfinite(got).all() and (err < tol).all(), (what, worst, err[worst], np.broadcast_to(tol, err.shape)[worst])


def chunk_tolerance(a, proj, by_head=False):
    """What operands of fp16 may do to the rows of a prompt from an empty state: four standard deviations, and the result's rounding.  A weight
    y^(i-j) (q . k) has the errors of q and k, which meet in sqrt(sum q^2 k^2), and its own; a value has one more.  Whole rows, or every head of them."""
    q, k, v, _ = a.heads(proj, 0)
    age = np.arange(len(proj))[:, None] - np.arange(len(proj))[None]
    errors, sizes = [], []
    for h in range(a.H):
        with np.errstate(invalid="ignore"):
            keep = np.where(age >= 0, np.where(age == 0, 1.0, np.exp(np.maximum(age, 1) * float(a.rates[h]))), 0.0)
        s, mag = q[:, h] @ k[:, h].T, np.sqrt((q[:, h] ** 2) @ (k[:, h] ** 2).T)
        scale = float(np.float32(a.cfg["scale"]))
        o = scale * (keep * s) @ v[:, h]
        err = 2.0 ** -12 * np.sqrt(2 / 3) * scale * np.sqrt((keep ** 2 * (mag ** 2 + s ** 2)) @ (v[:, h] ** 2).mean(axis=1))
        size = np.sqrt((o ** 2).mean(axis=1))
        f = 1 / np.sqrt(size ** 2 + a.eps) if a.norm is not None else 1.0
        errors.append((f * err) ** 2)
        sizes.append((f * size) ** 2)
    errors, sizes = np.array(errors).T, np.array(sizes).T
    return 2.0 ** -8 + 4 * np.sqrt(errors / sizes if by_head else errors.sum(axis=1) / sizes.sum(axis=1))


def states_near(a, slot):
    """fp32 sums (see states_close), every head beside its own largest number."""
    got, want, n = f64(a.states[slot]), a.memory[slot]["S"], a.memory[slot]["at"]
    for h in range(a.H):
        assert np.abs(got[h] - want[h]).max() <= 5 * np.sqrt(2 * n / 12) * 2.0 ** -23 * np.abs(want[h]).max(), h


def scale_tables(a, factor):
    """Rotary tables times a factor, on the device and for the oracle (whose parts that turn are so much larger)."""
    cos, sin = tables(a.rot, a.capacity)
    for r in (a.rotation, a.m.rotation):
        r.rope_cos, r.rope_sin = a.b.f32(factor * cos), a.b.f32(factor * sin)
    heads, n = a.heads, a.rot["dims"]

    def scaled(proj, first):
        q, k, v, g = heads(proj, first)
        q[..., :n] *= factor
        k[..., :n] *= factor
        return q, k, v, g

    a.heads = scaled


def parts(a, proj):
    """Columns of keys and of values."""
    n = a.H * a.d
    return proj[:, n:2 * n], proj[:, 2 * n:3 * n]


RATES = [-0.01, -0.5, 0.0, -20.0]


@pytest.mark.parametrize("norm", [True, False])
@pytest.mark.parametrize("head_norm", [True, False])
@pytest.mark.parametrize("n,at,power,dim", [(128, 127, 20, 128), (200, 199, 24, 64), (200, 40, 24, 90), (128, 64, 20, 128)])
def test_decay_rows_that_do_not_see_a_large_token(cuda, stack_lib, norm, head_norm, n, at, power, dim):
    """A token whose value is 2^20 times the others' reaches the rows behind it, as long as they remember it, and no others."""
    a = Decay(cuda, stack_lib, cfgd(4, dim, 44, 0.1, gated=False, norm=norm), 1, norm=head_norm, rates=RATES)
    proj = np.random.default_rng(n + at).standard_normal((n, a.cols)).astype(np.float32)
    parts(a, proj)[1][at] *= 2.0 ** power
    if not norm:
        parts(a, proj)[0][at] *= 2.0 ** 6
    tol, want = chunk_tolerance(a, proj), a.oracle([1], proj)
    own_rows_close(a.forward(CHUNK, [1], proj), want, tol, "rows")
    states_near(a, 1)


@pytest.mark.parametrize("norm", [True, False])
@pytest.mark.parametrize("power", [-16, -20, -30])
def test_decay_tokens_of_zeros_among_small_ones(cuda, stack_lib, norm, power):
    """Rows of zeros (padding, say) change nothing for the others, however small those are."""
    a = Decay(cuda, stack_lib, cfgd(4, 128, 64, 0.1, gated=False, norm=norm), 1, norm=False, rates=RATES)
    proj = np.random.default_rng(-power).standard_normal((200, a.cols)).astype(np.float32)
    parts(a, proj)[1][:] *= 2.0 ** power
    if not norm:
        parts(a, proj)[0][:] *= 2.0 ** power
    proj[[3, 70, 150]] = 0
    proj[[5, 71], :] *= np.float32(1e-3)
    parts(a, proj)[0][90] = 0                                   # a key alone
    parts(a, proj)[1][160] = 0                                  # a value alone
    rows = np.setdiff1d(np.arange(200), [3, 70, 150])           # (no query: zeros)
    with np.errstate(invalid="ignore"):
        tol, want = chunk_tolerance(a, proj)[rows], a.oracle([1], proj)
    got = a.forward(CHUNK, [1], proj)
    own_rows_close(got[rows], want[rows], tol, "rows")
    assert (got[[3, 70, 150]] == 0).all()
    states_near(a, 1)


def uneven(a, which, power):
    """Weights of the norm `which`: 2^power times as large in the first eight dimensions (a turning pair has both or neither)."""
    half = a.rot["dims"] // 2 if a.rot else 0
    w = getattr(a, which).copy()
    w[np.r_[0:4, half:half + 4]] *= np.float32(2.0 ** power)
    setattr(a, which, w)
    for r in (a.rotation, a.m.rotation):
        setattr(r, which, a.b.f32(w))


@pytest.mark.parametrize("dim", [128, 64, 90])
def test_decay_dimensions_of_very_different_sizes(cuda, stack_lib, dim):
    """Keys large where queries are small, values with one number far above the others: no number is lost beside a large one."""
    a = Decay(cuda, stack_lib, cfgd(3, dim, 44, 0.1, gated=False), 1, rates=[-0.01, -0.001, -0.3])
    uneven(a, "k_norm", 17)
    uneven(a, "q_norm", -17)
    proj = np.random.default_rng(dim).standard_normal((300, a.cols)).astype(np.float32)
    parts(a, proj)[1][:, 5::dim] *= 2.0 ** 18
    # every head by itself: its norm is that of its large number, whose error the others of the head share beside their own (a head whose large number is small
    # by chance has large others, of a large error)
    tol, want = chunk_tolerance(a, proj, by_head=True).ravel(), a.oracle([1], proj).reshape(-1, dim)
    got = a.forward(CHUNK, [1], proj).reshape(-1, dim)
    own_rows_close(got[:, 5:6], want[:, 5:6], tol, "the large numbers")
    rest = np.r_[0:5, 6:dim]
    own_rows_close(got[:, rest], want[:, rest], 2 * tol, "the others")


@pytest.mark.parametrize("norm", [True, False])
def test_decay_queries_far_below_the_norms_epsilon(cuda, stack_lib, norm):
    a = Decay(cuda, stack_lib, cfgd(3, 128, 64, 0.1, gated=False, norm=norm), 1, norm=False, rates=[-0.01, -0.001, -0.3])
    proj = np.random.default_rng(2).standard_normal((200, a.cols)).astype(np.float32)
    proj[10:190, :3 * 128] *= np.exp2(-np.arange(180) / 8).astype(np.float32)[:, None]
    tol, want = chunk_tolerance(a, proj), a.oracle([1], proj)
    own_rows_close(a.forward(CHUNK, [1], proj), want, tol, "rows")


@pytest.mark.parametrize("norm", [True, False])
def test_decay_with_tables_that_scale(cuda, stack_lib, norm):
    """Tables may hold more than cosines and sines: a factor of 16, say."""
    a = Decay(cuda, stack_lib, cfgd(3, 128, 64, 0.1, gated=False, norm=norm), 1, rates=[-0.01, -0.001, -0.3])
    scale_tables(a, 16)
    proj = np.random.default_rng(3).standard_normal((200, a.cols)).astype(np.float32)
    tol, want = chunk_tolerance(a, proj), a.oracle([1], proj)
    own_rows_close(a.forward(CHUNK, [1], proj), want, tol, "rows")


@pytest.mark.parametrize("precision,route,n", [(0, SIMT, 3), (1, SIMT, 3), (1, STREAM, 1), (1, STREAM, 3), (1, FLASH, 80)])
@pytest.mark.parametrize("gap", [8.0, 14.0, 16.0, 18.0, 20.0])
@pytest.mark.parametrize("place", [0, 40, 510])
def test_quantized_weights_beside_one_that_takes_nearly_everything(cuda, stack_lib, precision, route, n, gap, place):
    """A key far above the others whose value is zero: the output is the others' small sum.  Weights e^-gap of the largest, which in fp16 stand at 2^11 or above: at
    e^-20 = 2^-28.9 half a step of 2^-24 is 2^-7.1 of them (standard deviation 2^-7.9, many tokens), beside the result's 2^-8; in fp32 the 2e-5 of other tests."""
    a = Quantized(cuda, stack_lib, cfg4(4, 2, 64, 0, 1.0, gated=False, norm=False), precision, capacity=700)
    rng = np.random.default_rng(int(gap) + place)
    T, d, G = 600, 64, 2
    proj = rng.standard_normal((T + n, a.cols)).astype(np.float32)
    keys, values = proj[:, 4 * d:6 * d], proj[:, 6 * d:8 * d]
    sign = np.where(rng.random(2 * d) < 0.5, -1, 1)
    keys *= 2.0 ** -5
    keys[place], values[place] = 0.5 * sign, 0
    held = O.four_bits(keys[place].reshape(G, d), a.cfg["key_scale"])
    for h in range(4):                                           # queries along that key
        c = np.float16(gap / np.abs(held[h // 2]).sum())
        proj[:, h * d:(h + 1) * d] = c * sign[h // 2 * d:(h // 2 + 1) * d]
    before, rows = proj[:T], proj[T:]
    a.forward(SIMT, [1], before)
    a.oracle([1], before)
    want, got = a.oracle([1], rows), a.forward(route, [1], rows)
    own_rows_close(got.reshape(-1, d), want.reshape(-1, d), 2.0 ** -7 if precision else 2e-5, "heads")


@pytest.mark.parametrize("precision,route", [(0, SIMT), (0, 0), (1, SIMT), (1, STREAM), (1, FLASH), (1, 0)])
@pytest.mark.parametrize("before", [0, 32, 63, 128, 224, 300])
@pytest.mark.parametrize("what", ["key", "value"])
def test_quantized_numbers_that_are_not_finite_reach_the_rows_behind(cuda, stack_lib, precision, route, before, what):
    """A NaN in a key or value is seen in every head that reads it, also where it is the only token of a tile that a row sees, and in no other."""
    a = Quantized(cuda, stack_lib, cfg4(4, 2, 64, 32, 0.2, gated=False), precision)
    rng = np.random.default_rng(before)
    if before:
        a.forward(SIMT, [1], rng.standard_normal((before, a.cols)).astype(np.float32))
    d = 64
    proj = rng.standard_normal((1, a.cols)).astype(np.float32)
    proj[0, (5 if what == "key" else 7) * d + 3] = np.nan       # of key/value head 1
    for _ in range(3):                                           # the token itself, and two behind it
        got = a.forward(route, [1], proj).reshape(4, d)
        assert np.isfinite(got[:2]).all()
        assert np.isnan(got[2:]).all() if what == "key" else np.isnan(got[2:, :16]).all() and np.isfinite(got[2:, 16:]).all()
        proj = rng.standard_normal((1, a.cols)).astype(np.float32)


Q_CALLS = [(0, SIMT, 3), (1, SIMT, 3), (1, STREAM, 1), (1, STREAM, 3), (1, FLASH, 80)]


@pytest.mark.parametrize("precision,route,n", Q_CALLS)
@pytest.mark.parametrize("case", ["uneven", "uneven the other way", "far below epsilon", "tables that scale"])
def test_quantized_queries_of_very_different_sizes(cuda, stack_lib, precision, route, n, case):
    """No number of a query is lost beside a larger one, or under what its norm would allow.  Scores have a standard deviation s of some units; fp16 queries move
    one by 2^-12 / sqrt(3) s, and an output by about as much of itself: with s below 4, 2^-11, beside the result's 2^-8."""
    uneven_by = {"uneven": 18, "uneven the other way": -18}.get(case, 0)
    scale = {"far below epsilon": 6e4, "tables that scale": 0.2 / 256}.get(case, 0.3)
    units = (2.0 ** 9 if uneven_by > 0 else 0.5 if case == "tables that scale" else 0.05, 0.07)
    a = Quantized(cuda, stack_lib, cfg4(4, 2, 64, 64, scale, gated=False, units=units), precision, capacity=500)
    if uneven_by:
        uneven(a, "k_norm", uneven_by)
        uneven(a, "q_norm", -uneven_by)
    if case == "tables that scale":
        scale_tables(a, 16)
    rng = np.random.default_rng(len(case))
    proj = rng.standard_normal((400 + n, a.cols)).astype(np.float32)
    if case == "far below epsilon":
        proj[:, :4 * 64] *= np.float32(1e-7)
    before, rows = proj[:400], proj[400:]
    a.forward(SIMT, [1], before)
    a.oracle([1], before)
    want, got = a.oracle([1], rows), a.forward(route, [1], rows)
    own_rows_close(got.reshape(-1, 64), want.reshape(-1, 64), 2.0 ** -7 if precision else 2e-5, "heads")


@pytest.mark.parametrize("precision,route,n,dim", [(0, 0, 1, 64), (0, 0, 4, 128), (0, SCAN, 9, 64), (0, SCAN, 9, 90), (0, SCAN, 9, 256), (1, 0, 2, 128), (1, SCAN, 9, 128), (1, CHUNK, 9, 128),
                                                   (1, CHUNK, 2, 64)])
def test_decay_fast_decays_of_what_is_left(cuda, stack_lib, precision, route, n, dim):
    """After a token come ones without key or value (padding, say), which only read: what fast decays leave of the state keeps its bits, as little as it is.
    Six tokens' decays are off by three half steps each (two units in the last place of exp, a rounding), all of them together as one exponential by 48 x 2^-24 of its
    argument and two units: 4e-6."""
    rates = [-0.3, -0.49, -0.51, -0.7, -2.0, -5.0, -8.0]
    a = Decay(cuda, stack_lib, cfgd(len(rates), dim, 0, 0.1, gated=False, norm=False), precision, norm=False, rates=rates)
    rng = np.random.default_rng(n)
    proj = rng.standard_normal((n, a.cols)).astype(np.float32)
    a.forward(route, [1], proj)
    a.oracle([1], proj)
    left = 6
    while left:
        take = min(left, n)
        proj = rng.standard_normal((take, a.cols)).astype(np.float32)
        for p in parts(a, proj):
            p[:] = 0
        queries = a.heads(proj, a.memory[1]["at"])[0]
        want, got = a.oracle([1], proj), a.forward(route, [1], proj)
        # S q: four standard deviations of the operands' roundings (chunks: fp16) or of some ten fp32 ones, where its terms cancel as they do
        S = a.memory[1]["S"]
        o, size = (np.sqrt((np.einsum("hvk,thk->thv", x, y) ** p).mean(axis=2)) for x, y, p in ((S, queries, 2), (S ** 2, queries ** 2, 1)))
        step = (2.0 ** -12 * np.sqrt(2 / 3) if route == CHUNK else 2.0 ** -24 * np.sqrt(10)) * size / o
        own_rows_close(got.reshape(-1, dim), want.reshape(-1, dim), (4 * step + (2.0 ** -8 if precision else 0) + 4e-6).ravel(), "rows")
        left -= take
    got, want = f64(a.states[1]), a.memory[1]["S"]
    for h in range(a.H):
        assert np.abs(got[h] - want[h]).max() <= 4e-6 * np.abs(want[h]).max() + (5 * np.sqrt(2 * n / 12) * 2.0 ** -23) * np.abs(want[h]).max(), a.rates[h]


@pytest.mark.parametrize("precision,route,dim", [(0, SCAN, 64), (0, SCAN, 90), (1, SCAN, 128), (1, CHUNK, 128), (1, CHUNK, 90)])
@pytest.mark.parametrize("zeros", [40, 128, 200])
def test_decay_of_a_state_over_padding(cuda, stack_lib, precision, route, dim, zeros):
    """A prompt behind which as many tokens of zeros follow as leave e^-45 of its state, in one call (segments, chunks): the argument's rounding 45 x 2^-24, two units of
    exp for each of its up to three factors, a rounding each token (scan: the decay's own, at most 2^-23, too): 200 x 2^-23 at most."""
    rates = [-45.0 / zeros, -20.0 / zeros, -2.0 / zeros]
    a = Decay(cuda, stack_lib, cfgd(3, dim, 0, 0.1, gated=False, norm=False), precision, norm=False, rates=rates)
    rng = np.random.default_rng(zeros)
    proj = rng.standard_normal((100 + zeros, a.cols)).astype(np.float32)
    for p in parts(a, proj):
        p[100:] = 0
    a.oracle([1], proj)
    a.forward(route, [1], proj)
    got, want = f64(a.states[1]), a.memory[1]["S"]
    for h in range(a.H):
        assert np.abs(got[h] - want[h]).max() <= 200 * 2.0 ** -23 * np.abs(want[h]).max(), a.rates[h]
