"""4-bit attention where its routes change over: single tokens of short and long contexts, every place of a long history, many sequences at once; operators'
calls that the model tests reach only inside a stack."""
import numpy as np
import pytest

from oracle import layer_stack as O
from rotated_helpers import Decay, Quantized, stream
from test_gpu_rotated_mixers import FLASH, FOUR, SIMT, STREAM, cfg4, cfgd, states_close

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _built(cuda, stack_lib):
    stack_lib.tbl_device_status(stream(cuda))
    yield
    assert stack_lib.tbl_device_status(stream(cuda)) == 0


def own_rows_close(got, want, tol, what):
    err = np.sqrt(((got - want) ** 2).mean(axis=1)) / np.sqrt((want ** 2).mean(axis=1))
    assert np.isfinite(got).all() and err.max() < tol, (what, int(err.argmax()), err.max())


def shifted(a, proj):
    """The projections on the device, four bytes off a boundary of 16."""
    flat = a.torch.zeros(proj.size + 1, device="cuda")
    flat[1:] = a.device(proj).flatten()
    a.b.keep.append(flat)
    return flat[1:].view(proj.shape)


@pytest.mark.parametrize("shift", [False, True])
@pytest.mark.parametrize("precision,route", [(1, STREAM), (1, 0), (0, 0)])
@pytest.mark.parametrize("size", ["plain", "small", "odd", "dim192", "wide", "group12"])
def test_quantized_first_tokens(cuda, stack_lib, precision, route, size, shift):
    """Single tokens from the first one of an empty cache on, two sequences at different places, by the call that does everything in one launch (up to 128 tokens by
    four warps); rows that nobody has written hold NaNs.  An average of few values keeps their size, so a row is held to its own: rounding of the result 2^-8 (bf16)."""
    a = Quantized(cuda, stack_lib, FOUR[size], precision, slots=4, capacity=160)
    rng = np.random.default_rng(6)
    at = {1: 0, 3: 0}
    for first, second in [(0, 0), (1, 5), (31, 32), (33, 62), (63, 126), (127, 127), (128, 130)]:
        for slot, place in ((1, first), (3, second)):            # histories up to there
            if place > at[slot]:
                part = rng.standard_normal((place - at[slot], a.cols)).astype(np.float32)
                a.oracle([slot], part)
                a.forward(SIMT, [slot], part)
                at[slot] = place
        # one sequence alone (its context decides on the route), then both
        for slots in ([1], [3, 1]):
            proj = rng.standard_normal((len(slots), a.cols)).astype(np.float32)
            got = a.forward(route, slots, proj, pd=shifted(a, proj) if shift else None)
            own_rows_close(got, a.oracle(slots, proj), 2.0 ** -7 if precision else 2e-5, (first, second, slots))
            for s in slots:
                at[s] += 1
    for s in (1, 3):
        k, v = a.read(s, 0, at[s])
        np.testing.assert_allclose(k, np.array(a.memory[s][0]), rtol=2.0 ** -23, atol=0)
        np.testing.assert_allclose(v, np.array(a.memory[s][1]), rtol=2.0 ** -23, atol=0)
        assert bool((a.cache[s, :, at[s]:] == 255).all())
    assert bool((a.cache[[0, 2]] == 255).all())


@pytest.mark.parametrize("precision,route,n", [(0, SIMT, 3), (1, SIMT, 3), (1, STREAM, 1), (1, STREAM, 3), (1, FLASH, 80)])
def test_quantized_finds_every_place_of_a_long_history(cuda, stack_lib, precision, route, n):
    """A query aimed at one key finds its value: at tiles' and splits' borders, and at 240 places in between."""
    cfg = cfg4(4, 2, 64, 0, 1.0, gated=False, norm=False)
    T = 3000
    a = Quantized(cuda, stack_lib, cfg, precision, slots=2, capacity=T + 300)
    rng = np.random.default_rng(3)
    proj = rng.standard_normal((T, a.cols)).astype(np.float32)
    proj[:, :4 * 64] = 0
    a.forward(SIMT, [1], proj)
    keys, values = a.read(1, 0, T)
    places = np.r_[0, 1, 15, 16, 31, 32, 63, 64, 127, 128, T - 1, T - 2, rng.integers(0, T, 228)]
    for lo in range(0, 240, n):
        aimed = np.zeros((n, a.cols), np.float32)
        aimed[:, 4 * 64:] = rng.standard_normal((n, a.cols - 4 * 64)) * 1e-3
        for h in range(4):
            key = keys[places[lo:lo + n], h // 2]
            aimed[:, h * 64:(h + 1) * 64] = key * (200.0 / (key * key).sum(axis=1, keepdims=True))
        got = a.forward(route, [1], aimed, advance=False).reshape(n, 4, 64)
        for t in range(n):
            for h in range(4):
                want = values[places[lo + t], h // 2]
                # in fp32 a number is the value but for a few roundings (other keys have e^-40 of the weight and less)
                assert np.abs(got[t, h] - want).max() <= (2.0 ** -7 if precision else 2e-5) * np.abs(want).max(), (places[lo + t], h)


@pytest.mark.parametrize("precision,route,n,T,size", [(1, STREAM, 1, 3000, "plain"), (1, STREAM, 3, 3000, "plain"), (1, STREAM, 2, 7001, "group12"), (1, STREAM, 1, 9000, "odd"),
                                                      (1, 0, 1, 2000, "small"), (1, STREAM, 4, 2500, "wide"), (0, 0, 1, 5000, "plain"), (0, SIMT, 3, 2500, "wide"), (1, FLASH, 130, 2000, "odd")])
def test_quantized_long_history_with_weights_spread_out(cuda, stack_lib, precision, route, n, T, size):
    """Thousands of tokens that all count, over splits of the context.  A row is held to its own size; the average of T values of random sign is a small number, and so are
    its errors: those of the weights (2^-12, at random) as of the result (2^-8)."""
    a = Quantized(cuda, stack_lib, FOUR[size], precision, slots=2, capacity=T + 300)
    rng = np.random.default_rng(T)
    for lo in range(0, T, 1000):
        part = rng.standard_normal((min(1000, T - lo), a.cols)).astype(np.float32)
        a.forward(SIMT, [1], part)
        q, k, v, _ = a.heads(part, lo)                           # (the oracle's history, without its outputs)
        memory = a.memory.setdefault(1, ([], []))
        memory[0].extend(O.four_bits(k, a.cfg["key_scale"]))
        memory[1].extend(O.four_bits(v, a.cfg["value_scale"]))
    for _ in range(2):
        proj = rng.standard_normal((n, a.cols)).astype(np.float32)
        own_rows_close(a.forward(route, [1], proj), a.oracle([1], proj), 2.0 ** -7 if precision else 2e-5, "rows")


@pytest.mark.parametrize("precision,heads,kv,dim,seqs", [(1, 8, 2, 64, 160), (1, 4, 4, 128, 80), (0, 4, 2, 40, 170), (1, 2, 1, 256, 310)])
def test_quantized_tokens_of_many_sequences(cuda, stack_lib, precision, heads, kv, dim, seqs):
    """More sequences and heads than the GPU takes at once: the call of one launch gives way to two."""
    a = Quantized(cuda, stack_lib, cfg4(heads, kv, dim, dim // 4 * 2, 0.2), precision, slots=seqs + 1, capacity=70)
    rng = np.random.default_rng(seqs)
    slots = (rng.permutation(seqs) + 1).tolist()
    part = rng.standard_normal((seqs * 37, a.cols)).astype(np.float32)
    a.forward(SIMT, slots, part)
    a.oracle(slots, part)
    more = rng.standard_normal((seqs // 3 * 28, a.cols)).astype(np.float32)     # a third of them are further on
    a.forward(0, slots[:seqs // 3], more)
    a.oracle(slots[:seqs // 3], more)
    for n in (1, 1, 2):
        proj = rng.standard_normal((seqs * n, a.cols)).astype(np.float32)
        own_rows_close(a.forward(0, slots, proj), a.oracle(slots, proj), 2.0 ** -7 if precision else 2e-5, n)
    assert bool((a.cache[0] == 255).all())


@pytest.mark.parametrize("dim,gated", [(220, True), (224, True), (256, False), (216, False), (66, True), (130, False)])
@pytest.mark.parametrize("precision", [0, 1])
def test_decay_single_tokens_of_heads_that_do_not_fit_one_launch(cuda, stack_lib, precision, dim, gated):
    """Heads of 224 and more (four tokens: 216), or not a multiple of four, take the scan also for single tokens."""
    a = Decay(cuda, stack_lib, cfgd(3, dim, 32, 0.1, gated=gated), precision)
    rng = np.random.default_rng(dim)
    for slots, n in [([1], 1), ([2], 4), ([1, 2], 1), ([2, 1], 2), ([1], 3), ([1, 2], 4), ([1, 2], 1)]:
        proj = rng.standard_normal((len(slots) * n, a.cols)).astype(np.float32)
        own_rows_close(a.forward(0, slots, proj), a.oracle(slots, proj), 2.0 ** -7 if precision else 2e-5, (slots, n))
        states_close(a, slots)
    assert not bool(a.states[0].any())
