"""Normed and rotated heads, 4-bit cache, decay attention: how they are called -- one norm of two, other numbers of tokens, two calls at once, captured
calls, prompts in several pieces, rows far into a large cache, far more heads than a block takes."""
import ctypes as C

import numpy as np
import pytest

from rotated_helpers import Buf, Decay, Quantized, f64, fp32_rotation, stream, tables
from test_gpu_rotated_mixers import CHUNK, DECAY, FLASH, FOUR, SCAN, SIMT, STREAM, cfg4, cfgd, rows_close, states_close

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _built(cuda, stack_lib):
    stack_lib.tbl_device_status(stream(cuda))
    yield
    assert stack_lib.tbl_device_status(stream(cuda)) == 0


def without(a, which):
    """Takes one of the two norms away."""
    setattr(a, which, None)
    setattr(a.m.rotation, which, None)
    return a


@pytest.mark.parametrize("which", ["q_norm", "k_norm"])
@pytest.mark.parametrize("precision,route", [(0, SIMT), (1, STREAM), (1, FLASH)])
def test_quantized_with_one_norm(cuda, stack_lib, which, precision, route):
    a = without(Quantized(cuda, stack_lib, cfg4(6, 2, 128, 96, 0.05, units=(0.3, 0.4)), precision), which)
    rng = np.random.default_rng(8)
    for slots, n in [([1], 70), ([2], 49), ([1, 2], 3), ([2, 1], 1)]:
        proj = rng.standard_normal((len(slots) * n, a.cols)).astype(np.float32)
        rows_close(a.forward(route, slots, proj), a.oracle(slots, proj), 2.0 ** -7 if precision else 2e-5, (slots, n))


@pytest.mark.parametrize("which", ["q_norm", "k_norm"])
@pytest.mark.parametrize("precision,route", [(0, SCAN), (1, SCAN), (1, CHUNK)])
def test_decay_with_one_norm(cuda, stack_lib, which, precision, route):
    a = without(Decay(cuda, stack_lib, cfgd(3, 128, 96, 0.05), precision), which)
    rng = np.random.default_rng(8)
    for slots, n in [([1], 150), ([2], 64), ([1, 2], 3), ([2, 1], 1)]:
        proj = rng.standard_normal((len(slots) * n, a.cols)).astype(np.float32)
        rows_close(a.forward(route, slots, proj), a.oracle(slots, proj), 2.0 ** -7 if precision else 2e-5, (slots, n))
        states_close(a, slots)


@pytest.mark.parametrize("which", [0, 1])
def test_rotation_with_one_norm_and_many_heads(cuda, stack_lib, which):
    """Query and key heads share warps; 300 + 20 heads are more than one round of a block."""
    from reimagined_b200 import capi
    torch, b, rng, P, H, G, d, eps = cuda, Buf(cuda), np.random.default_rng(4), 64, 300, 20, 48, 1e-3
    cfg = {"base": 50.0, "dims": 16, "interleaved": True}
    w = (1 + 0.2 * rng.standard_normal(d)).astype(np.float32)
    norms = [None, None]
    norms[which] = w
    r = capi.HeadRotation(*(None if x is None else b.f32(x) for x in norms), *[b.f32(t) for t in tables(cfg, P)], 16, P, 1)
    x = (3 * rng.standard_normal((5, (H + G) * d))).astype(np.float32)
    q, k = (torch.zeros((5, c, d), device="cuda") for c in (H, G))
    assert stack_lib.tbl_head_rotation_forward(C.byref(r), 0, eps, b.f32(x), (H + G) * d, H, G, d, b.i32([0]), b.i32([7]), 1, 5, q.data_ptr(), k.data_ptr(), stream(torch)) == 0
    for got, lo, count, norm in ((q, 0, H, norms[0]), (k, H * d, G, norms[1])):
        want = fp32_rotation(x[:, lo:lo + count * d].reshape(5, count, d), norm, cfg, np.arange(7, 12), eps)
        size = np.sqrt((want ** 2).mean(axis=-1, keepdims=True))
        assert (np.abs(f64(got) - want) <= 16 * 2.0 ** -24 * (np.abs(want) + 4 * size)).all()


@pytest.mark.parametrize("precision", [0, 1])
@pytest.mark.parametrize("size", ["plain", "small", "odd", "tiny", "dim200", "wide"])
def test_decay_between_a_few_tokens_and_a_prompt(cuda, stack_lib, precision, size):
    a = Decay(cuda, stack_lib, DECAY[size], precision)
    rng = np.random.default_rng(12)
    for slots, n in [([1], 9), ([1, 2], 20), ([2], 8), ([1], 47), ([2, 1], 33), ([1], 64), ([2], 65), ([1], 257)]:
        proj = rng.standard_normal((len(slots) * n, a.cols)).astype(np.float32)
        rows_close(a.forward(SCAN if n > 47 else 0, slots, proj), a.oracle(slots, proj), 2.0 ** -7 if precision else 2e-5, (slots, n))
        states_close(a, slots)


@pytest.mark.parametrize("seqs,heads,n", [(64, 4, 517), (100, 4, 300)])
def test_decay_prompts_in_pieces(cuda, stack_lib, seqs, heads, n):
    """So many sequences that the chunks' operands pass what one piece holds; against the scan, which has no pieces.  Outputs of either are bf16 (half a step each:
    2^-8 together) of sums that agree to fp16 operands; states are fp32 sums that may round every token once more."""
    torch = cuda
    a = Decay(cuda, stack_lib, cfgd(heads, 128, 64, 0.1), 1, slots=seqs)
    a.positions += 3
    proj = torch.randn((seqs * n, a.cols), device="cuda", generator=torch.Generator("cuda").manual_seed(3))
    slots = torch.randperm(seqs, generator=torch.Generator().manual_seed(1)).tolist()
    a.states.copy_(torch.randn(a.states.shape, device="cuda", generator=torch.Generator("cuda").manual_seed(4)))
    outs, states = [], []
    for route in (SCAN, CHUNK):
        into = torch.full_like(a.states, 9.0)
        outs.append(a.forward(route, slots, proj, advance=False, into=into, pd=proj))
        states.append(into.double())
    rows_close(outs[1], outs[0], 2.0 ** -7, "outputs")
    assert float((states[0] - states[1]).abs().max()) <= 2 * 5 * np.sqrt(2 * n / 12) * 2.0 ** -23 * float(states[0].abs().max())


def captured(torch, call, outs):
    """The call's results, the same from a replay on another stream."""
    assert call() == 0
    first = [o.clone() for o in outs]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        assert call() == 0
    for o in outs:
        o.zero_()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        graph.replay()
        graph.replay()
    side.synchronize()
    for a, b in zip(first, outs):
        assert torch.equal(a, b)


# one token whole, one token of a long context (splits, or sixteen warps), several tokens, a portion, fp32
@pytest.mark.parametrize("precision,route,n,before,size", [(1, 0, 1, 300, "plain"), (1, 0, 1, 3000, "plain"), (1, STREAM, 3, 3000, "group12"), (1, 0, 64, 300, "plain"), (1, FLASH, 64, 300, "plain"),
                                                           (0, 0, 2, 900, "odd"), (1, 0, 1, 700, "wide")])
def test_quantized_captured(cuda, stack_lib, precision, route, n, before, size):
    torch = cuda
    a = Quantized(cuda, stack_lib, FOUR[size], precision, slots=2, capacity=before + n)
    rng = np.random.default_rng(2)
    a.forward(0, [1], rng.standard_normal((before, a.cols)).astype(np.float32))
    proj = a.device(rng.standard_normal((n, a.cols)))
    out = torch.zeros((n, a.H * a.d), device="cuda", dtype=a.dtype)
    bytes_ = stack_lib.tbl_quantized_workspace_bytes(C.byref(a.m), precision, route, 1, n, before + n)
    ws, slots = a.space(bytes_), a.b.i32([1])
    captured(torch, lambda: stack_lib.tbl_quantized_forward(C.byref(a.m), precision, route, a.eps, proj.data_ptr(), a.cache.data_ptr(), 2, a.capacity, slots, a.positions.data_ptr(),
                                                            1, n, before + n, out.data_ptr(), ws.data_ptr(), bytes_, stream(torch)), [out])


@pytest.mark.parametrize("precision,route,n,size", [(0, 0, 301, "odd"), (1, CHUNK, 130, "small"), (1, 0, 20, "plain"), (1, 0, 1, "plain")])
def test_decay_captured(cuda, stack_lib, precision, route, n, size):
    torch = cuda
    a = Decay(cuda, stack_lib, DECAY[size], precision, slots=2)
    rng = np.random.default_rng(2)
    a.forward(0, [1], rng.standard_normal((70, a.cols)).astype(np.float32))
    proj, into = a.device(rng.standard_normal((n, a.cols))), torch.zeros_like(a.states)
    out = torch.zeros((n, a.H * a.d), device="cuda", dtype=a.dtype)
    bytes_ = stack_lib.tbl_decay_workspace_bytes(C.byref(a.m), precision, route, 1, n)
    ws, slots = a.space(bytes_), a.b.i32([1])
    captured(torch, lambda: stack_lib.tbl_decay_forward(C.byref(a.m), precision, route, a.eps, proj.data_ptr(), a.states.data_ptr(), into.data_ptr(), slots, a.positions.data_ptr(),
                                                        1, n, out.data_ptr(), ws.data_ptr(), bytes_, stream(torch)), [out, into])


@pytest.mark.parametrize("kind,n", [("decay", 300), ("decay", 2), ("four", 1), ("four", 90)])
def test_two_calls_at_once(cuda, stack_lib, kind, n):
    """Two streams, each with its own state and workspace, give the bits that each gives alone."""
    torch = cuda
    make = (lambda: Decay(cuda, stack_lib, DECAY["plain"], 1, slots=1, capacity=3000)) if kind == "decay" else (lambda: Quantized(cuda, stack_lib, FOUR["plain"], 1, slots=1, capacity=3000))
    rng = np.random.default_rng(9)
    both = [rng.standard_normal((p, make().cols)).astype(np.float32) for p in (500, 500)]
    steps = [[rng.standard_normal((n, both[0].shape[1])).astype(np.float32) for _ in range(6)] for _ in both]

    def run(together):
        objects, outs = [make() for _ in both], [[], []]
        for a, p in zip(objects, both):
            a.forward(0, [0], p)
        steps_d = [[a.device(x) for x in s] for a, s in zip(objects, steps)]
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in both]
        keep = []
        for i in range(6):
            for j, a in enumerate(objects):
                with torch.cuda.stream(streams[j]):
                    out = torch.zeros((n, a.H * a.d), device="cuda", dtype=a.dtype)
                    if kind == "decay":
                        size = stack_lib.tbl_decay_workspace_bytes(C.byref(a.m), 1, 0, 1, n)
                        keep.append(a.space(size))
                        rc = stack_lib.tbl_decay_forward(C.byref(a.m), 1, 0, a.eps, steps_d[j][i].data_ptr(), a.states.data_ptr(), a.states.data_ptr(), a.b.i32([0]),
                                                         a.positions.data_ptr(), 1, n, out.data_ptr(), keep[-1].data_ptr(), size, stream(torch))
                    else:
                        size = stack_lib.tbl_quantized_workspace_bytes(C.byref(a.m), 1, 0, 1, n, 3000)
                        keep.append(a.space(size))
                        rc = stack_lib.tbl_quantized_forward(C.byref(a.m), 1, 0, a.eps, steps_d[j][i].data_ptr(), a.cache.data_ptr(), 1, a.capacity, a.b.i32([0]),
                                                             a.positions.data_ptr(), 1, n, 3000, out.data_ptr(), keep[-1].data_ptr(), size, stream(torch))
                    assert rc == 0
                    a.positions += n
                    outs[j].append(out)
                if not together:
                    torch.cuda.synchronize()
        torch.cuda.synchronize()
        return outs, [a.states if kind == "decay" else a.cache for a in objects]

    alone, held = run(False)
    at_once, held2 = run(True)
    for x, y in zip(alone[0] + alone[1] + held, at_once[0] + at_once[1] + held2):
        assert torch.equal(x, y)


@pytest.mark.parametrize("precision,route,n", [(0, SIMT, 2), (1, STREAM, 1), (1, FLASH, 64)])
def test_quantized_cache_past_32_bits(cuda, stack_lib, precision, route, n):
    """A slot of more than 2^31 bytes: a query finds a key that lies millions of tokens back, and its token is written at the far end."""
    torch = cuda
    cap = 8_000_000
    a = Quantized(cuda, stack_lib, cfg4(4, 2, 128, 0, 1.0, gated=False, norm=False), precision, slots=2, capacity=cap)
    assert a.G * cap * a.row > 2 ** 31
    a.cache[1].zero_()                                   # keys and values of zero
    rng = np.random.default_rng(6)
    planted = rng.standard_normal((1, a.cols)).astype(np.float32)
    for place in (cap - 5000, 5, cap - 70):
        a.positions[1] = place
        a.forward(SIMT, [1], planted, advance=False)
    keys, values = a.read(1, cap - 5000, 1)
    a.positions[1] = cap - n
    proj = np.zeros((n, a.cols), np.float32)
    for h in range(4):
        key = keys[0, h // 2]
        proj[:, h * 128:(h + 1) * 128] = key * (200.0 / (key @ key))
    got = a.forward(route, [1], proj, advance=False).reshape(n, 4, 128)
    for h in range(4):                                   # three copies of the same key: the same value
        want = values[0, h // 2]
        assert np.abs(got[:, h] - want).max() <= (2.0 ** -7 if precision else 2e-5) * np.abs(want).max()
    far = a.cache[1, :, cap - n:]
    assert not bool(far.any()) and bool((a.cache[0] == 255).all())               # the new tokens' keys and values are zero too


@pytest.mark.parametrize("precision,route,n", [(0, SIMT, 3), (1, STREAM, 1), (1, STREAM, 3), (1, FLASH, 64)])
def test_quantized_norms_written_by_the_call_ahead(cuda, stack_lib, precision, route, n):
    """Norms are operands like any other: the call before may have written them.  (Here a rotation without angles, which copies fp32 heads.)"""
    from reimagined_b200 import capi
    torch = cuda
    a = Quantized(cuda, stack_lib, cfg4(4, 2, 64, 32, 0.2), precision)
    rng = np.random.default_rng(4)
    proj = rng.standard_normal((n, a.cols)).astype(np.float32)
    pd, out = a.device(proj), torch.zeros((n, a.H * a.d), device="cuda", dtype=a.dtype)
    norms, big = torch.zeros((2, 64), device="cuda"), torch.zeros((4096, 4096), device="cuda")
    for m in (a.rotation, a.m.rotation):
        m.q_norm, m.k_norm = norms[0].data_ptr(), norms[1].data_ptr()
    size = stack_lib.tbl_quantized_workspace_bytes(C.byref(a.m), precision, route, 1, n, n)
    ws, zero, plain = a.space(size), a.b.i32([0]), capi.HeadRotation()
    for _ in range(20):
        a.q_norm, a.k_norm = (1 + 0.2 * rng.standard_normal(64).astype(np.float32) for _ in range(2))
        source = a.device([a.q_norm, a.k_norm])
        a.memory.clear()
        want = a.oracle([0], proj)
        big.fill_(1.0)                                           # keeps the stream busy until everything is enqueued
        assert stack_lib.tbl_head_rotation_forward(C.byref(plain), 0, a.eps, source.data_ptr(), 64, 1, 0, 64, zero, zero, 1, 2, norms.data_ptr(), None, stream(torch)) == 0
        assert stack_lib.tbl_quantized_forward(C.byref(a.m), precision, route, a.eps, pd.data_ptr(), a.cache.data_ptr(), 3, a.capacity, zero, a.positions.data_ptr(), 1, n, n,
                                               out.data_ptr(), ws.data_ptr(), size, stream(torch)) == 0
        rows_close(f64(out), want, 2.0 ** -7 if precision else 2e-5, "rows")
