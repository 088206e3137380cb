"""Normed and rotated heads, attention over a 4-bit cache and linear attention with decay, through the C ABI, against float64.

Tolerances.  A bf16 result is its value rounded once: half a step, 2^-8 of it, beside what its operands were rounded to before.
fp32: sums of at most 2^9 products and a few operations on them, 2^-24 each, random in sign: 2e-5 of a row's size is 300 of them."""
import ctypes as C

import numpy as np
import pytest

from oracle import layer_stack as O
from rotated_helpers import Buf, Decay, Quantized, f64, fp32_rotation, stream, tables

pytestmark = pytest.mark.gpu
SIMT, STREAM, FLASH = 1, 2, 3
SCAN, CHUNK = 1, 2
FULL = 4


@pytest.fixture(scope="module", autouse=True)
def _built(cuda, stack_lib):
    stack_lib.tbl_device_status(stream(cuda))
    yield
    assert stack_lib.tbl_device_status(stream(cuda)) == 0


def rows_close(got, want, tol, what):
    """Every row's error against the rows' usual size (a row may be the small difference of large terms, whose rounding it keeps)."""
    err = np.sqrt(((got - want) ** 2).mean(axis=1)) / np.sqrt((want ** 2).mean())
    assert np.isfinite(got).all() and err.max() < tol, (what, int(err.argmax()), err.max())


# ---- heads ----------------------------------------------------------------------------------------------------------------
HEADS = [  # query heads, key heads, dim, rotated, interleaved, norm
    (32, 8, 128, 128, False, True), (4, 4, 64, 64, False, True), (3, 1, 256, 256, True, True), (2, 5, 128, 64, True, True), (6, 2, 80, 32, False, True),
    (1, 0, 128, 128, False, True), (0, 3, 96, 96, True, True), (5, 2, 90, 44, False, True), (5, 2, 37, 10, True, True), (2, 2, 1, 0, False, True),
    (2, 1, 2, 2, True, True), (7, 3, 255, 254, False, True), (4, 2, 128, 0, False, True), (4, 2, 64, 24, False, False), (80, 8, 128, 128, False, True),
    (3, 2, 33, 0, False, False)]


@pytest.mark.parametrize("precision", [0, 1])
@pytest.mark.parametrize("H,G,d,rot,pairs,norm", HEADS)
@pytest.mark.parametrize("seqs,n,gap,shift", [(1, 1, 0, 0), (3, 5, 12, 0), (2, 170, 0, 0), (2, 3, 5, 1)])
def test_head_rotation(cuda, stack_lib, precision, H, G, d, rot, pairs, norm, seqs, n, gap, shift):
    from reimagined_b200 import capi
    torch, b, rng, P, eps = cuda, Buf(cuda), np.random.default_rng(H * d + n), 300, 1e-3
    cfg = {"base": 50.0, "dims": rot, "interleaved": pairs} if rot else None
    wq, wk = ((1 + 0.2 * rng.standard_normal(d)).astype(np.float32) if norm else None for _ in range(2))
    r = capi.HeadRotation(b.f32(wq) if norm else None, b.f32(wk) if norm else None, *([b.f32(t) for t in tables(cfg, P)] if rot else [None, None]), rot, P if rot else 0,
                          int(pairs))
    ld, rows = (H + G) * d + gap, seqs * n
    x = (rng.standard_normal((rows, ld)) * 3).astype(np.float32)
    flat = torch.zeros(rows * ld + shift, device="cuda")
    flat[shift:] = torch.as_tensor(x).cuda().flatten()
    slots, begin = rng.permutation(seqs + 2)[:seqs], np.zeros(seqs + 2, int)
    begin[slots] = rng.integers(0, P - n, seqs)
    dtype = torch.bfloat16 if precision else torch.float32
    q, k = (torch.full((rows, c, d), 7.0, device="cuda", dtype=dtype) for c in (H, G))
    rc = stack_lib.tbl_head_rotation_forward(C.byref(r), precision, eps, flat.data_ptr() + 4 * shift, ld, H, G, d, b.i32(slots), b.i32(begin), seqs, n,
                                             q.data_ptr() if H else None, k.data_ptr() if G else None, stream(torch))
    assert rc == 0
    at = np.concatenate([np.arange(begin[s], begin[s] + n) for s in slots])
    for got, lo, count, w in ((q, 0, H, wq), (k, H * d, G, wk)):
        if count:
            want = fp32_rotation(x[:, lo:lo + count * d].reshape(rows, count, d), w, cfg, at, eps)
            size = np.sqrt((want ** 2).mean(axis=-1, keepdims=True)) + 1e-30
            # a rounding to bf16, and a dozen fp32 operations of the size of the pair
            assert (np.abs(f64(got) - want) <= (2.0 ** -8 * np.abs(want) if precision else 0) + 16 * 2.0 ** -24 * (np.abs(want) + 4 * size)).all()


def test_head_rotation_leaves_rows_beyond_the_tables(cuda, stack_lib):
    from reimagined_b200 import capi
    torch, b, d = cuda, Buf(cuda), 64
    cfg = {"base": 50.0, "dims": 64}
    r = capi.HeadRotation(None, None, *[b.f32(t) for t in tables(cfg, 10)], 64, 10, 0)
    x = np.random.default_rng(0).standard_normal((6, 2 * d)).astype(np.float32)
    q, k = (torch.full((6, 1, d), 7.0, device="cuda") for _ in range(2))
    call = lambda begin: stack_lib.tbl_head_rotation_forward(C.byref(r), 0, 0.0, b.f32(x), 2 * d, 1, 1, d, b.i32([0, 1]), b.i32(begin), 2, 3, q.data_ptr(), k.data_ptr(),
                                                             stream(torch))
    assert call([7, 8]) == 0
    assert stack_lib.tbl_device_status(stream(torch)) & FULL
    assert bool((q[5] == 7).all()) and bool((k[5] == 7).all()) and not bool((q[:5] == 7).any())
    assert call([-1, 0]) == 0
    assert stack_lib.tbl_device_status(stream(torch)) & FULL


# ---- 4-bit cache -----------------------------------------------------------------------------------------------------------
def cfg4(heads, kv, dim, rot, scale, pairs=False, gated=True, norm=True, units=(0.05, 0.07)):
    return {"heads": heads, "kv_heads": kv, "dim": dim, "scale": scale, "key_scale": units[0], "value_scale": units[1], "qk_norm": norm, "gated": gated,
            "rot": {"base": 300.0, "dims": rot, "interleaved": pairs} if rot else None}


FOUR = {
    "plain": cfg4(8, 2, 128, 128, 0.2),
    "small": cfg4(4, 4, 64, 64, 0.3, gated=False),
    "odd": cfg4(10, 2, 90, 44, 0.2, pairs=True),
    "tiny": cfg4(3, 1, 5, 4, 0.7),
    "wide": cfg4(2, 1, 256, 64, 0.1),
    "dim192": cfg4(6, 2, 192, 192, 0.1, gated=False),
    "group12": cfg4(12, 1, 128, 64, 0.15, pairs=True),
    "group20": cfg4(40, 2, 64, 0, 0.2),
    "raw": cfg4(6, 3, 72, 24, 0.05, norm=False, units=(0.3, 1.7)),
}
Q_ROUTES = [SIMT, STREAM, FLASH]


@pytest.mark.parametrize("precision,route,size", [(0, SIMT, s) for s in FOUR] + [(1, r, s) for r in Q_ROUTES for s in FOUR if (r, s) != (FLASH, "wide")] + [(0, 0, "odd"), (1, 0, "plain"), (1, 0, "odd")])
def test_quantized_attention(cuda, stack_lib, precision, route, size):
    """A prompt in portions, then single tokens, on two slots at different places; rows behind the sequences hold NaNs throughout."""
    a = Quantized(cuda, stack_lib, FOUR[size], precision)
    rng = np.random.default_rng(5)
    # bf16: the result's rounding (2^-9 of its size on the average at most, 2^-8 of the largest numbers); the flash kernel's queries are rounded too
    tol = 2.0 ** -7 if precision else 2e-5
    for slots, n in [([1], 130), ([1], 2), ([2], 61), ([1, 2], 3), ([1, 2], 1), ([2, 1], 1), ([1, 2], 140), ([2], 1)]:
        proj = rng.standard_normal((len(slots) * n, a.cols)).astype(np.float32)
        rows_close(a.forward(route, slots, proj), a.oracle(slots, proj), tol, f"slots {slots} n {n}")
    assert bool((a.cache[0] == 255).all()) and bool((a.cache[1, :, int(a.positions[1]):] == 255).all())       # nobody touched those
    for slot, (keys, values) in a.memory.items():
        k, v = a.read(slot, 0, len(keys))
        np.testing.assert_allclose(k, np.array(keys), rtol=2.0 ** -23, atol=0)
        np.testing.assert_allclose(v, np.array(values), rtol=2.0 ** -23, atol=0)
    assert stack_lib.tbl_device_status(stream(cuda)) == 0


def test_quantized_flash_refuses_heads_it_has_no_room_for(cuda, stack_lib):
    a = Quantized(cuda, stack_lib, FOUR["wide"], 1)
    a.forward(FLASH, [1], np.zeros((60, a.cols), np.float32), check_rc=-2)
    assert bool((a.cache == 255).all())


def test_quantized_numbers(cuda, stack_lib):
    """Ties, zeros, ends of the scales, numbers that are not finite."""
    cfg = cfg4(1, 1, 64, 0, 0.1, gated=False, norm=False, units=(0.5, 2.0 ** -3))
    a = Quantized(cuda, stack_lib, cfg, 0)
    steps = np.array([0.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -0.25, -0.75, -1.25, -1.75, -2.5, -3.5, -5.0, 6.0])
    rows = []
    for unit in (0.5, 2.0 ** -3):
        group = [steps * unit * f for f in (1.0, 2.0, 0.125, 448.0)]             # ties between codes, exact scales
        rows.append(np.concatenate(group))
    big, small = np.full(64, 1e30), np.full(64, 1e-12)
    bad = np.ones(64)
    bad[[3, 20, 40]] = np.nan, np.inf, -np.inf
    between = np.concatenate([np.r_[np.zeros(15), 6 * 0.5 * s] for s in (1.0625, 1.1875, 2.0 ** -10, 3 * 2.0 ** -10)])    # ties between scales
    x = np.stack([np.concatenate([np.zeros(64), k, v]) for k, v in [(rows[0], rows[1]), (big, small), (small, big), (bad, bad), (between, between), (np.zeros(64), -rows[1])]])
    a.forward(SIMT, [1], x.astype(np.float32))
    k, v = a.read(1, 0, 6)
    np.testing.assert_array_equal(k[:, 0], O.four_bits(x[:, 64:128], 0.5))
    np.testing.assert_array_equal(v[:, 0], O.four_bits(x[:, 128:], 2.0 ** -3))
    # 16 ones: s = e4m3(1 / 3) = 0.34375, 1 / (0.5 s) = 5.8 is code 6, 6 x 0.34375 x 0.5 = 1.03125
    assert np.isnan(k[3, 0, :48]).all() and (k[3, 0, 48:] == 1.03125).all() and k[1, 0, 0] == 448 * 6 * 0.5 and (v[1] == 0).all()
    k16, _ = a.read(1, 0, 6, 1)
    np.testing.assert_array_equal(k16, k)                                        # bf16 holds them where the unit is a power of two


@pytest.mark.parametrize("precision,route", [(0, SIMT), (1, SIMT), (1, STREAM), (1, FLASH)])
def test_quantized_finds_keys_far_back(cuda, stack_lib, precision, route):
    """A query aimed at one key of a long history finds its value, wherever the key lies against tiles and splits."""
    cfg = cfg4(4, 2, 64, 0, 1.0, gated=False, norm=False)
    T = 3000
    a = Quantized(cuda, stack_lib, cfg, precision, slots=2, capacity=T + 300)
    rng = np.random.default_rng(3)
    proj = rng.standard_normal((T, a.cols)).astype(np.float32)
    proj[:, :4 * 64] = 0
    a.forward(FLASH if precision else SIMT, [1], proj)
    keys, values = a.read(1, 0, T)
    for first in (0, 200):
        places = rng.integers(0, T, 160)
        places[:12] = 0, 1, 15, 16, 31, 32, 63, 64, 127, 128, T - 1, T - 2
        n = 3 if route == STREAM else 80
        aimed = np.zeros((n, a.cols), np.float32)
        aimed[:, 4 * 64:] = rng.standard_normal((n, a.cols - 4 * 64)) * 1e-3
        for lo in range(0, 12, n):
            for t in range(n):
                for h in range(4):
                    key = keys[places[lo + t], h // 2]
                    aimed[t, h * 64:(h + 1) * 64] = key * (200.0 / (key @ key))
            got = a.forward(route, [1], aimed, advance=False).reshape(n, 4, 64)
            for t in range(n):
                for h in range(4):
                    want = values[places[lo + t], h // 2]
                    assert np.abs(got[t, h] - want).max() <= 2.0 ** -7 * np.abs(want).max(), (places[lo + t], h)


@pytest.mark.parametrize("route", [SIMT, STREAM, FLASH])
def test_quantized_reports_a_full_cache(cuda, stack_lib, route):
    a = Quantized(cuda, stack_lib, FOUR["plain"], 1, slots=3, capacity=64)
    rng = np.random.default_rng(1)
    proj = rng.standard_normal((2 * 50, a.cols)).astype(np.float32)
    want = a.oracle([0, 2], proj)
    got = a.forward(route, [0, 2], proj)
    rows_close(got, want, 2.0 ** -7, "before")
    before = a.cache.clone()
    a.positions[2] = 62
    # the sequence in slot 2 has room for two of its three tokens; the other is not disturbed
    more = rng.standard_normal((2 * 3, a.cols)).astype(np.float32)
    want = a.oracle([0], more[:3])
    n = 3
    out = cuda.zeros((6, a.H * a.d), device="cuda", dtype=a.dtype)
    size = stack_lib.tbl_quantized_workspace_bytes(C.byref(a.m), 1, route, 2, n, 64)
    ws, pd = a.space(size), a.device(more)
    assert stack_lib.tbl_quantized_forward(C.byref(a.m), 1, route, a.eps, pd.data_ptr(), a.cache.data_ptr(), 3, 64, a.b.i32([0, 2]), a.positions.data_ptr(), 2, n, 64,
                                           out.data_ptr(), ws.data_ptr(), size, stream(cuda)) == 0
    rows_close(f64(out)[:3], want, 2.0 ** -7, "the other sequence")
    assert stack_lib.tbl_device_status(stream(cuda)) & FULL
    assert bool((a.cache[1] == before[1]).all()) and bool((a.cache[2, :, :62] == before[2, :, :62]).all()) and not bool((a.cache[2, :, 62:] == 255).all())


def test_quantized_repeated_call_and_other_stream(cuda, stack_lib):
    """The same call twice gives the same bits; so does a replayed capture on another stream."""
    torch = cuda
    a = Quantized(cuda, stack_lib, FOUR["plain"], 1, slots=2)
    rng = np.random.default_rng(2)
    a.forward(0, [0], rng.standard_normal((200, a.cols)).astype(np.float32))
    proj = a.device(rng.standard_normal((1, a.cols)))
    out, n = torch.zeros((1, a.H * a.d), device="cuda", dtype=a.dtype), 1
    size = stack_lib.tbl_quantized_workspace_bytes(C.byref(a.m), 1, 0, 1, n, 256)
    ws, slots = a.space(size), a.b.i32([0])
    call = lambda: stack_lib.tbl_quantized_forward(C.byref(a.m), 1, 0, a.eps, proj.data_ptr(), a.cache.data_ptr(), 2, a.capacity, slots, a.positions.data_ptr(), 1, n, 256,
                                                   out.data_ptr(), ws.data_ptr(), size, stream(torch))
    assert call() == 0
    first = out.clone()
    assert call() == 0 and torch.equal(first, out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        assert call() == 0
    out.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(first, out)
    a.positions += 1                                  # the replay goes by the positions on the device
    a.memory[0] = None
    graph.replay()
    torch.cuda.synchronize()
    assert not torch.equal(first, out) and bool(torch.isfinite(out).all())


# ---- decay -----------------------------------------------------------------------------------------------------------------
def states_close(a, slots):
    """fp32 sums of the tokens so far: two roundings a token, each a random number of at most half a step of 2^-23 of the largest of the state (standard deviation
    2^-23 / sqrt(12)), five standard deviations of their sum."""
    for s in slots:
        got, want, n = f64(a.states[s]), a.memory[s]["S"], a.memory[s]["at"]
        for h in range(a.H):
            assert np.abs(got[h] - want[h]).max() <= 5 * np.sqrt(2 * n / 12) * 2.0 ** -23 * np.abs(want[h]).max(), (s, h)


def cfgd(heads, dim, rot, scale, pairs=False, gated=True, norm=True):
    return {"heads": heads, "dim": dim, "scale": scale, "gated": gated, "qk_norm": norm, "rot": {"base": 300.0, "dims": rot, "interleaved": pairs} if rot else None}


DECAY = {
    "plain": cfgd(3, 128, 128, 0.1),
    "small": cfgd(4, 64, 64, 0.2, gated=False),
    "odd": cfgd(2, 90, 44, 0.15, pairs=True),
    "tiny": cfgd(2, 5, 2, 0.5),
    "raw": cfgd(2, 72, 24, 0.1, norm=False),
    "one": cfgd(1, 1, 0, 1.0),
    "wide": cfgd(2, 256, 64, 0.1),
    "dim200": cfgd(1, 200, 0, 0.1, gated=False),
}
C_SIZES = [s for s in DECAY if s not in ("wide", "dim200")]


@pytest.mark.parametrize("precision,route,size", [(0, SCAN, s) for s in DECAY] + [(1, SCAN, "plain"), (1, SCAN, "odd"), (1, SCAN, "wide")] +
                         [(1, CHUNK, s) for s in C_SIZES] + [(1, 0, "plain"), (1, 0, "odd"), (0, 0, "small")])
def test_decay_attention(cuda, stack_lib, precision, route, size):
    """Prompts in portions and single tokens, on two slots at different places."""
    a = Decay(cuda, stack_lib, DECAY[size], precision)
    rng = np.random.default_rng(5)
    tol = 2.0 ** -7 if precision else 2e-5
    if size == "one" and route == CHUNK:
        # A head of one number may come out near zero, where its norm has the slope 1 / sqrt(eps): that times the rounding of the terms (three operands of
        # about one, 2^-12 each at most) of as many tokens as the decay keeps, which add up at random: four standard deviations.
        tol += 4 * 2.0 ** -12 * np.sqrt(3 / (1 - np.exp(2.0 * a.rates.max()))) / np.sqrt(a.eps)
    for slots, n in [([1], 130), ([1], 2), ([2], 61), ([1, 2], 3), ([1, 2], 1), ([2, 1], 1), ([1, 2], 270), ([2], 1), ([1, 2], 128), ([2], 129)]:
        proj = rng.standard_normal((len(slots) * n, a.cols)).astype(np.float32)
        rows_close(a.forward(route, slots, proj), a.oracle(slots, proj), tol, f"slots {slots} n {n}")
        states_close(a, slots)
    assert not bool(a.states[0].any())
    assert stack_lib.tbl_device_status(stream(cuda)) == 0


@pytest.mark.parametrize("precision,route", [(0, SCAN), (1, SCAN), (1, CHUNK)])
def test_decay_forgets_and_remembers(cuda, stack_lib, precision, route):
    """No memory at all, a token's, no decay, a decay that fp32 can hardly tell from none; no head norm; states into another array."""
    rates = [-np.inf, -200.0, -1.0, -1e-3, -1e-6, 0.0]
    a = Decay(cuda, stack_lib, cfgd(6, 64, 32, 0.1), precision, norm=False, rates=rates)
    rng = np.random.default_rng(6)
    for slots, n in [([0, 2], 300), ([0, 2], 1), ([0, 2], 700)]:
        proj = rng.standard_normal((len(slots) * n, a.cols)).astype(np.float32)
        into = cuda.full_like(a.states, 3.0)
        before = a.states.clone()
        got = a.forward(route, slots, proj, into=into)
        want = a.oracle(slots, proj)
        rows_close(got, want, 2.0 ** -7 if precision else 2e-5, n)
        assert cuda.equal(before, a.states) and bool((into[1] == 3).all())
        into[1] = 0
        a.states = into
        states_close(a, slots)


@pytest.mark.parametrize("precision,n", [(1, 8), (1, 300), (0, 20)])
def test_decay_repeated_call_and_capture(cuda, stack_lib, precision, n):
    torch = cuda
    a = Decay(cuda, stack_lib, DECAY["plain"], precision, slots=2)
    rng = np.random.default_rng(2)
    a.forward(0, [1], rng.standard_normal((70, a.cols)).astype(np.float32))
    proj, into = a.device(rng.standard_normal((n, a.cols))), torch.zeros_like(a.states)
    out = torch.zeros((n, a.H * a.d), device="cuda", dtype=a.dtype)
    size = stack_lib.tbl_decay_workspace_bytes(C.byref(a.m), precision, 0, 1, n)
    ws, slots = a.space(size), a.b.i32([1])
    call = lambda: stack_lib.tbl_decay_forward(C.byref(a.m), precision, 0, a.eps, proj.data_ptr(), a.states.data_ptr(), into.data_ptr(), slots, a.positions.data_ptr(), 1, n,
                                               out.data_ptr(), ws.data_ptr(), size, stream(torch))
    assert call() == 0
    first, state = out.clone(), into.clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        assert call() == 0
    out.zero_()
    into.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(first, out) and torch.equal(state, into)


def test_decay_reports_positions_beyond_the_tables(cuda, stack_lib):
    a = Decay(cuda, stack_lib, DECAY["plain"], 1, capacity=100)
    proj = np.random.default_rng(0).standard_normal((2 * 60, a.cols)).astype(np.float32)
    a.positions[1] = 70
    a.memory[0] = {"at": 0, "S": np.zeros((a.H, a.d, a.d))}
    got = a.forward(0, [0, 1], proj)
    assert stack_lib.tbl_device_status(stream(cuda)) & FULL
    rows_close(got[:60], a.oracle([0], proj[:60]), 2.0 ** -7, "the other sequence")


# ---- models ----------------------------------------------------------------------------------------------------------------
def model(layers, width, vocab=97):
    import stack_helpers as S
    return S.config(layers, width, vocab)


def decay_layer(*args, mlp=None, **kw):
    return {"type": "decay_attention", "mixer": cfgd(*args, **kw), "mlp": mlp}


def four_layer(*args, mlp=None, **kw):
    return {"type": "quantized_attention", "mixer": cfg4(*args, **kw), "mlp": mlp}


def models():
    import stack_helpers as S
    return {
        "decay": model([decay_layer(3, 64, 32, 0.2, mlp=S.ff(96)), decay_layer(2, 90, 44, 0.1, pairs=True, norm=False), S.delta(2, 40)], 128),
        "four": model([four_layer(8, 2, 64, 64, 0.2, mlp=S.ff(96)), four_layer(4, 4, 40, 20, 0.2, pairs=True, gated=False)], 128),
        "mixed": model([decay_layer(2, 128, 128, 0.1), four_layer(4, 1, 128, 64, 0.1, mlp=S.ff(72)), decay_layer(4, 32, 0, 0.2, gated=False)], 136),
    }


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name", ["decay", "four", "mixed"])
def test_models_with_these_mixers(cuda, stack_lib, name, dtype):
    """Prompts, portions, tokens decoded together by captured steps, slots used again: one model against the oracle.

    4-bit codes amplify: borders are some 0.4 of a number's standard deviation s apart, so bf16 activations (2^-8 s off) put 2 x 2^-8 / 0.4 = 2 % of the numbers
    on the other side of one, each 0.4 s off: sqrt(0.02) x 0.4 = 6 % of a token's values, which a first token passes on unaveraged, twice (two such
    layers): 0.12.  fp32 moves none or one of a row of 512 and more: 0.4 / sqrt(512) = 2 %."""
    import stack_helpers as S
    from oracle.layer_stack import decoder
    from reimagined_b200.stack import StackEngine, synthetic_weights
    cfg = models()[name]
    w = synthetic_weights(cfg, 3, 8)
    p = {k: v.float().numpy().astype(np.float64) for k, v in w.items()}
    e = StackEngine(cfg, w, dtype, slots=3, capacity=400)
    rng = np.random.default_rng(1)
    ids = [rng.integers(0, 97, 170).tolist() for _ in range(2)]
    want = [decoder(cfg, p).feed(i) for i in ids]
    limit = (4e-2, 2e-5) if name == "decay" else (0.12, 2e-2)
    limit = limit[dtype == "float32"]
    for _ in range(2):                                   # the second time in slots that were used
        slots = [e.open(), e.open()]
        got = e.feed(slots[0], ids[0][:120], list(range(120)))
        assert S.row_errors(got, want[0][:120]).max() <= limit
        got = e.feed(slots[1], ids[1][:7], list(range(7)))
        got = e.feed(slots[1], ids[1][7:70], list(range(63)))
        assert S.row_errors(got, want[1][7:70]).max() <= limit
        for t in range(12):
            got = e.step(slots, [[ids[0][120 + t]], [ids[1][70 + t]]])
            assert S.row_errors(got, np.stack([want[0][120 + t], want[1][70 + t]])).max() <= limit, t
        got = e.step(slots, [ids[0][132:135], ids[1][82:85]], want=list(range(6)))
        assert S.row_errors(got, np.concatenate([want[0][132:135], want[1][82:85]])).max() <= limit
        for s in slots:
            e.close(s)
    assert e.device_status() == 0
