"""Head rotation, 4-bit cache and decay attention: what needs no GPU -- the oracle by hand, configurations, refusals."""
import ctypes as C

import numpy as np
import pytest
import torch

from oracle import layer_stack as O


def test_oracle_rotation_of_neighbours():
    x = np.arange(1.0, 9.0)[None, None]
    y = O.rotate_pairs(x, [3], 10.0, 6)
    a = 3 * 10.0 ** (-2 / 6)                                    # the second pair: entries 2 and 3
    np.testing.assert_allclose(y[0, 0, 2:4], [3 * np.cos(a) - 4 * np.sin(a), 4 * np.cos(a) + 3 * np.sin(a)])
    np.testing.assert_allclose(y[0, 0, 6:], x[0, 0, 6:])


def test_oracle_four_bits_by_hand():
    # largest 12, unit 1: scale e4m3(2) = 2; 5 / 2 = 2.5 lies between 2 and 3, the even code is 2; 0.5 / 2 = 0.25 between 0 and 0.5
    x = np.zeros(16)
    x[:5] = 12, -5, 0.5, 0.51, 7
    np.testing.assert_array_equal(O.four_bits(x, 1.0)[:5], [12, -4, 0, 1, 8])
    # scales end at 448: 448 x 6
    assert O.four_bits(np.full(16, 1e9), 1.0)[0] == 448 * 6 and (O.four_bits(np.full(16, 1e-9), 1.0) == 0).all()
    assert np.isnan(O.four_bits(np.r_[np.inf, np.zeros(15)], 1.0)).all()
    assert O.four_bits(np.arange(20.0), 1.0).shape == (20,)
    got = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    np.testing.assert_array_equal(O.E4M3, got)


def test_oracle_decay_by_hand():
    cfg, eye = {"heads": 1, "dim": 1, "scale": 2.0}, np.eye(1)
    P = {"q": eye, "k": 3 * eye, "v": -eye, "decay": [np.log(np.log(2.0))], "norm": [1.0], "o": eye}         # S <- S / 2 + v k
    m = {"tokens": 0, "states": np.zeros((1, 1, 1))}
    O.decay_attention(np.array([[1.0], [2.0]]), P, "", cfg, 1e-3, m)
    np.testing.assert_allclose(m["states"], -3 / 2 - 12)
    assert m["tokens"] == 2


def rotated(**kw):
    from reimagined_b200 import capi
    d = dict(q_norm=4096, k_norm=4096, rope_cos=4096, rope_sin=4096, rot_dim=16, rope_positions=64, interleaved=0)
    d.update(kw)
    return capi.HeadRotation(*(d[n] for n, _ in capi.HeadRotation._fields_))


def test_head_rotation_refuses_before_it_touches_a_device(stack_lib):
    before = stack_lib.tbl_launch_count()
    call = lambda **k: stack_lib.tbl_head_rotation_forward(C.byref(k.get("r", rotated())), k.get("precision", 1), k.get("eps", 1e-5), k.get("proj", 4096), k.get("ld", 192),
                                                           k.get("q", 4), k.get("k", 2), k.get("dim", 32), k.get("slots", 4096), 4096, k.get("n_seq", 1), k.get("n_tok", 1),
                                                           k.get("q_dev", 4096), k.get("k_dev", 4096), None)
    for bad in (dict(proj=None), dict(slots=None), dict(precision=2), dict(q=-1), dict(q_dev=None), dict(k_dev=None), dict(n_seq=0), dict(n_tok=0), dict(q=0, k=0),
                dict(eps=float("nan")), dict(eps=-1.0), dict(r=rotated(rope_cos=None)), dict(r=rotated(rope_positions=0)), dict(r=rotated(interleaved=2))):
        assert call(**bad) == -1, bad
    for bad in (dict(dim=0), dict(dim=257, ld=10000), dict(ld=191), dict(r=rotated(rot_dim=34)), dict(r=rotated(rot_dim=15)), dict(n_seq=65536, n_tok=65536)):
        assert call(**bad) == -2, bad
    assert call(proj=4098) == -6
    assert stack_lib.tbl_launch_count() == before


def quantized(**kw):
    from reimagined_b200 import capi
    d = dict(heads=4, kv_heads=2, dim=32, gated=1, scale=0.2, key_scale=0.1, value_scale=0.1, rotation=rotated())
    d.update(kw)
    cols = (d["heads"] * (1 + d["gated"]) + 2 * d["kv_heads"]) * d["dim"]
    return capi.QuantizedMixer(capi.DenseView(4096, None, 8, kw.get("cols", cols)), capi.DenseView(4096, None, d["heads"] * d["dim"], 8), d["rotation"], d["heads"], d["kv_heads"],
                               d["dim"], d["gated"], d["scale"], d["key_scale"], d["value_scale"])


def test_factors_of_scores_and_outputs(stack_lib):
    before = stack_lib.tbl_launch_count()
    for scale in (0.0, -0.2, float("nan"), float("inf"), 1e38, 1e-38):
        assert stack_lib.tbl_quantized_forward(C.byref(quantized(scale=scale)), 1, 0, 1e-5, 4096, 4096, 2, 16, 4096, 4096, 1, 1, 16, 4096, 4096, 1 << 40, None) == -4
        assert stack_lib.tbl_quantized_workspace_bytes(C.byref(quantized(scale=scale)), 1, 0, 1, 1, 16) == 0
    m = decay()
    for m.scale in (float("nan"), float("inf")):
        assert stack_lib.tbl_decay_forward(C.byref(m), 1, 0, 1e-5, 4096, 4096, 4096, 4096, 4096, 1, 1, 4096, 4096, 1 << 40, None) == -4
    m.scale = -0.5
    assert stack_lib.tbl_decay_workspace_bytes(C.byref(m), 1, 0, 1, 1) > 0
    assert stack_lib.tbl_launch_count() == before


def test_results_lie_on_their_types_bytes(stack_lib):
    before = stack_lib.tbl_launch_count()
    for precision, q, k, rc in ((0, 4098, 4096, -6), (0, 4096, 4098, -6), (1, 4097, 4096, -6), (1, 4096, 4099, -6)):
        assert stack_lib.tbl_head_rotation_forward(C.byref(rotated()), precision, 1e-5, 4096, 192, 4, 2, 32, 4096, 4096, 1, 1, q, k, None) == rc
        assert stack_lib.tbl_quantized_read(C.byref(quantized()), precision, 4096, 2, 16, 4096, 4096, 1, 1, q, k, None) == rc
    assert stack_lib.tbl_launch_count() == before


def test_quantized_attention_refuses_before_it_touches_a_device(stack_lib):
    L, before = stack_lib, stack_lib.tbl_launch_count()
    call = lambda m=None, **k: L.tbl_quantized_forward(C.byref(m or quantized()), k.get("precision", 1), k.get("route", 0), 1e-5, k.get("proj", 4096), k.get("cache", 4096), 2, 16,
                                                       4096, 4096, k.get("n_seq", 1), k.get("n_tok", 1), k.get("context", 16), 4096, k.get("ws", 4096), k.get("bytes", 1 << 40), None)
    for bad in (dict(precision=2), dict(route=4), dict(route=-1), dict(proj=None), dict(cache=None), dict(n_seq=3), dict(n_tok=0), dict(context=17), dict(n_tok=9, context=8)):
        assert call(**bad) == -1, bad
    for bad in (dict(kv_heads=3), dict(dim=257), dict(dim=0), dict(cols=100), dict(rotation=rotated(rot_dim=34))):
        assert call(quantized(**bad)) == -2, bad
    for bad in (dict(key_scale=0.0), dict(value_scale=-1.0), dict(key_scale=float("nan")), dict(value_scale=float("inf"))):
        assert call(quantized(**bad)) == -4, bad
    assert call(bytes=0) == -7 and call(ws=4096 + 16) == -6 and call(cache=4096 + 8) == -6
    assert call(precision=0, route=2) == -2 and call(precision=0, route=3) == -2 and call(quantized(dim=256), route=3) == -2
    read = lambda m=None, **k: L.tbl_quantized_read(C.byref(m or quantized()), k.get("precision", 1), k.get("cache", 4096), 2, 16, 4096, 4096, 1, 1, k.get("keys", 4096),
                                                    k.get("values", 4096), None)
    assert read(keys=None, values=None) == -1 and read(cache=None) == -1 and read(precision=5) == -1 and read(cache=4104) == -6 and read(quantized(kv_heads=3)) == -2
    # a row: codes and scales of a head of 32, padded to 64, and to 16 bytes
    assert [L.tbl_quantized_row_bytes(C.byref(quantized(dim=d))) for d in (32, 64, 65, 128, 192, 256)] == [80, 80, 144, 144, 224, 288]
    assert L.tbl_quantized_row_bytes(C.byref(quantized(kv_heads=3))) == 0 and L.tbl_quantized_workspace_bytes(C.byref(quantized()), 1, 9, 1, 1, 16) == 0
    assert L.tbl_launch_count() == before


def decay(**kw):
    from reimagined_b200 import capi
    d = dict(heads=4, dim=32, gated=1, log_decay=4096, norm=4096, rotation=rotated())
    d.update(kw)
    return capi.DecayMixer(capi.DenseView(4096, None, 8, kw.get("cols", (3 + d["gated"]) * d["heads"] * d["dim"])), capi.DenseView(4096, None, d["heads"] * d["dim"], 8), d["rotation"],
                           d["log_decay"], d["norm"], d["heads"], d["dim"], d["gated"], 0.2)


def test_decay_attention_refuses_before_it_touches_a_device(stack_lib):
    L, before = stack_lib, stack_lib.tbl_launch_count()
    call = lambda m=None, **k: L.tbl_decay_forward(C.byref(m or decay()), k.get("precision", 1), k.get("route", 0), 1e-5, k.get("proj", 4096), k.get("states", 4096), k.get("next", 4096),
                                                   4096, 4096, k.get("n_seq", 1), k.get("n_tok", 1), k.get("out", 4096), k.get("ws", 4096), k.get("bytes", 1 << 40), None)
    for bad in (dict(precision=2), dict(route=3), dict(proj=None), dict(states=None), dict(next=None), dict(n_seq=0), dict(n_tok=0), dict(out=None)):
        assert call(**bad) == -1, bad
    assert call(decay(log_decay=None)) == -1 and call(decay(gated=2)) == -1
    for bad in (dict(heads=0), dict(dim=257), dict(cols=100), dict(rotation=rotated(rot_dim=40))):
        assert call(decay(**bad)) == -2, bad
    assert call(bytes=0) == -7 and call(ws=4096 + 16) == -6 and call(states=4100) == -6 and call(precision=0, route=2) == -2 and call(decay(dim=200), route=2) == -2
    assert L.tbl_launch_count() == before


def test_configurations_of_these_mixers():
    import stack_helpers as S
    from reimagined_b200.stack import check_weights, synthetic_weights
    rot = {"base": 100.0, "dims": 8}
    cfg = S.config([{"type": "quantized_attention", "mlp": None, "mixer": {"heads": 4, "kv_heads": 2, "dim": 16, "scale": 0.2, "key_scale": 0.1, "value_scale": 0.1, "rot": rot}},
                    {"type": "decay_attention", "mlp": S.ff(8), "mixer": {"heads": 3, "dim": 12, "scale": 0.2, "rot": None, "qk_norm": False, "gated": False}}], 32, 50)
    w = synthetic_weights(cfg, 1, 4)
    assert w["l0.mix.k"].shape == (32, 32) and w["l0.mix.q.norm"].shape == (16,) and w["l0.mix.g"].shape == (64, 32)
    assert w["l1.mix.decay"].shape == (3,) and "l1.mix.g" not in w and "l1.mix.q.norm" not in w
    check_weights(cfg, w)
    for change in (lambda d: d.pop("l0.mix.q.norm"), lambda d: d.update({"l1.mix.g": torch.zeros(36, 32)}), lambda d: d.update({"l1.mix.decay": torch.zeros(4)})):
        d = dict(w)
        change(d)
        with pytest.raises(ValueError):
            check_weights(cfg, d)


def test_state_of_these_layers(stack_lib):
    """A 4-bit cache is its rows, a decay layer its states, whatever the precision of the activations."""
    from reimagined_b200 import capi

    def size(layer, precision, slots=3, capacity=50):
        m = capi.StackModel(8, 100, 1, 4096, 1.0, 1e-5, C.pointer(layer), 4096, capi.DenseView(4096, None, 8, 100))
        return stack_lib.tbl_stack_state_bytes(C.byref(m), precision, slots, capacity)

    layer = capi.StackLayer()
    layer.mixer, layer.norm1, layer.quantized = capi.MIXER_QUANTIZED_ATTENTION, 4096, quantized()
    assert size(layer, 1) == size(layer, 0) == 256 + -(-3 * 50 * 2 * 80 // 256) * 256
    layer.mixer, layer.decay = capi.MIXER_DECAY_ATTENTION, decay()
    assert size(layer, 1) == size(layer, 0) == 256 + 3 * 4 * 32 * 32 * 4
    layer.decay.heads = 5
    assert size(layer, 1) == 0


def test_a_workspace_for_the_longest_serves_shorter_calls(stack_lib):
    """Whatever route a shorter context, or a shorter portion, takes."""
    L = stack_lib
    for heads, kv, dim in ((32, 8, 128), (8, 8, 64), (16, 1, 128), (12, 2, 192), (4, 2, 256)):
        m = quantized(heads=heads, kv_heads=kv, dim=dim, rotation=rotated(rot_dim=dim))
        for precision in (0, 1):
            for n_seq, n_tok in ((1, 1), (9, 1), (150, 1), (1, 5), (3, 64), (8, 192), (1, 600)):
                sizes = [L.tbl_quantized_workspace_bytes(C.byref(m), precision, 0, n_seq, n_tok, n_tok + extra) for extra in [*range(0, 3000, 37), 5000, 8000, 16000, 131000]]
                assert sizes[0] > 0 and sizes == sorted(sizes), (heads, dim, precision, n_seq, n_tok)
    for heads, dim in ((32, 128), (10, 90), (4, 64), (2, 256), (300, 64)):
        m = decay(heads=heads, dim=dim, rotation=rotated(rot_dim=2))
        for precision in (0, 1):
            for n_seq in (1, 3, 40):
                sizes = [L.tbl_decay_workspace_bytes(C.byref(m), precision, 0, n_seq, n) for n in [*range(1, 700), 1024, 4096, 4999, 5000, 5120, 8192]]
                assert sizes[0] > 0 and sizes == sorted(sizes), (heads, dim, precision, n_seq)


def test_more_query_rows_than_a_grid_has(stack_lib):
    """65536 blocks of sixteen rows: refused before anything is appended."""
    before, n, m = stack_lib.tbl_launch_count(), 4 << 16, quantized(heads=4, kv_heads=1)
    for precision, route in ((0, 0), (0, 1), (1, 1), (1, 2)):
        assert stack_lib.tbl_quantized_forward(C.byref(m), precision, route, 1e-5, 4096, 4096, 2, n, 4096, 4096, 1, n, n, 4096, 4096, 1 << 60, None) == -2
    assert stack_lib.tbl_launch_count() == before


def test_more_than_the_prompt_kernel_holds(stack_lib):
    """Heads in two parts that pass a grid's side, and expanded rows that pass 32 bits: refused before anything is appended."""
    before = stack_lib.tbl_launch_count()
    for m, n_seq, context in ((quantized(heads=32768, kv_heads=1, dim=136, gated=0), 1, 64), (quantized(heads=8, kv_heads=8), 64, 4194304), (quantized(heads=8, kv_heads=8), 64, 4194304 - 100)):
        assert stack_lib.tbl_quantized_forward(C.byref(m), 1, 3, 1e-5, 4096, 4096, 64, 4194304, 4096, 4096, n_seq, 64, context, 4096, 4096, (1 << 63) - 1, None) == -2
    assert stack_lib.tbl_launch_count() == before
