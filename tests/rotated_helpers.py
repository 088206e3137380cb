"""Mixers with normed and rotated heads, on given projections, beside the same in the oracle."""
import ctypes as C

import numpy as np

from oracle import layer_stack as O


class Buf:
    """Keeps tensors alive and hands out pointers."""

    def __init__(self, torch):
        self.torch, self.keep = torch, []

    def put(self, a, dtype):
        self.keep.append(self.torch.as_tensor(np.asarray(a, dtype)).cuda().contiguous())
        return self.keep[-1].data_ptr()

    def f32(self, a):
        return self.put(a, np.float32)

    def i32(self, a):
        return self.put(a, np.int32)


def stream(torch):
    return torch.cuda.current_stream().cuda_stream


def f64(t):
    return t.detach().float().cpu().numpy().astype(np.float64)


def tables(rot, positions):
    freq = float(rot["base"]) ** (-2.0 * np.arange(rot["dims"] // 2) / rot["dims"])
    angle = np.arange(positions)[:, None] * freq[None]
    return np.cos(angle), np.sin(angle)


def fp32_rotation(x, norm, rot, positions, eps):
    """The oracle's heads, with the rotation by the fp32 tables that the operators read."""
    x = np.asarray(x, np.float64) if norm is None else O.rms_norm(x, np.float32(norm), eps)
    if rot is None:
        return x
    cos, sin = (t.astype(np.float32).astype(np.float64)[positions][:, None] for t in tables(rot, max(positions) + 1))
    half, y = rot["dims"] // 2, x.copy()
    a, b = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if rot.get("interleaved") else (slice(0, half), slice(half, 2 * half))
    y[..., a], y[..., b] = x[..., a] * cos - x[..., b] * sin, x[..., b] * cos + x[..., a] * sin
    return y


class Rotated:
    """Common part: sizes of the stacked projections, norms, tables."""

    def __init__(self, torch, lib, cfg, precision, slots, capacity, eps, seed=7):
        from reimagined_b200 import capi
        self.torch, self.lib, self.cfg, self.precision, self.capacity, self.eps, self.n_slots = torch, lib, cfg, precision, capacity, eps, slots
        self.b, self.capi = Buf(torch), capi
        self.H, self.G, self.d, self.rot = cfg["heads"], cfg.get("kv_heads", cfg["heads"]), cfg["dim"], cfg.get("rot")
        self.gated = cfg.get("gated", True)
        rng = np.random.default_rng(seed)
        self.q_norm, self.k_norm = ((1 + 0.2 * rng.standard_normal(self.d)).astype(np.float32) if cfg.get("qk_norm", True) else None for _ in range(2))
        self.rotation = r = capi.HeadRotation()
        if self.q_norm is not None:
            r.q_norm, r.k_norm = self.b.f32(self.q_norm), self.b.f32(self.k_norm)
        if self.rot is not None:
            r.rot_dim, r.rope_positions, r.interleaved = self.rot["dims"], capacity, int(bool(self.rot.get("interleaved")))
            r.rope_cos, r.rope_sin = (self.b.f32(t) for t in tables(self.rot, capacity))
        self.cols = (self.H + 2 * self.G + self.H * self.gated) * self.d
        self.dtype = torch.bfloat16 if precision else torch.float32
        self.positions = torch.zeros(slots, dtype=torch.int32, device="cuda")
        self.dummy = self.b.put(np.zeros(16), np.float32)
        self.views = capi.DenseView(self.dummy, None, 8, self.cols), capi.DenseView(self.dummy, None, self.H * self.d, 8)

    def split(self, proj):
        proj = np.asarray(proj, np.float64)
        n, at = self.d, 0
        out = []
        for count in (self.H, self.G, self.G, self.H if self.gated else 0):
            out.append(proj[:, at:at + count * n].reshape(len(proj), count, n) if count else None)
            at += count * n
        return out

    def heads(self, proj, first):
        q, k, v, g = self.split(proj)
        at = np.arange(first, first + len(proj))
        return (fp32_rotation(q, self.q_norm, self.rot, at, self.eps), fp32_rotation(k, self.k_norm, self.rot, at, self.eps), v,
                None if g is None else g.reshape(len(proj), -1))

    def space(self, size):
        return self.torch.full((size,), 255, dtype=self.torch.uint8, device="cuda")         # NaN patterns: nothing unwritten may be used

    def device(self, proj):
        return self.torch.as_tensor(np.asarray(proj, np.float32)).cuda()


class Quantized(Rotated):
    """Attention over a 4-bit cache.  Rows that nobody has written hold NaNs."""

    def __init__(self, torch, lib, cfg, precision, slots=3, capacity=420, eps=1e-3, **kw):
        super().__init__(torch, lib, cfg, precision, slots, capacity, eps, **kw)
        self.m = self.capi.QuantizedMixer(*self.views, self.rotation, self.H, self.G, self.d, int(self.gated), cfg["scale"], cfg["key_scale"], cfg["value_scale"])
        self.row = lib.tbl_quantized_row_bytes(C.byref(self.m))
        self.cache = torch.full((slots, self.G, capacity, self.row), 255, dtype=torch.uint8, device="cuda")
        self.memory = {}

    def forward(self, route, slots, proj, check_rc=0, advance=True, pd=None):
        torch, n_seq = self.torch, len(slots)
        n = len(proj) // n_seq
        context = int(self.positions[slots].max()) + n
        out = torch.zeros((n_seq * n, self.H * self.d), device="cuda", dtype=self.dtype)
        size = self.lib.tbl_quantized_workspace_bytes(C.byref(self.m), self.precision, route, n_seq, n, context)
        ws = self.space(max(size, 256))
        pd = self.device(proj) if pd is None else pd
        rc = self.lib.tbl_quantized_forward(C.byref(self.m), self.precision, route, self.eps, pd.data_ptr(), self.cache.data_ptr(), self.n_slots,
                                            self.capacity, self.b.i32(slots), self.positions.data_ptr(), n_seq, n, context, out.data_ptr(),
                                            ws.data_ptr(), size, stream(torch))
        assert rc == check_rc
        if rc == 0 and advance:
            self.positions[slots] += n
        return f64(out)

    def read(self, slot, first, n, precision=0):
        torch, dtype = self.torch, self.torch.bfloat16 if precision else self.torch.float32
        k, v = (torch.zeros((n, self.G, self.d), device="cuda", dtype=dtype) for _ in range(2))
        at = torch.full((self.n_slots,), first, dtype=torch.int32, device="cuda")
        assert self.lib.tbl_quantized_read(C.byref(self.m), precision, self.cache.data_ptr(), self.n_slots, self.capacity, self.b.i32([slot]), at.data_ptr(), 1, n,
                                           k.data_ptr(), v.data_ptr(), stream(torch)) == 0
        return f64(k), f64(v)

    def oracle(self, slots, proj):
        n, outs = len(proj) // len(slots), []
        for i, s in enumerate(slots):
            part = proj[i * n:(i + 1) * n]
            keys, values = self.memory.setdefault(s, ([], []))
            first = len(keys)
            q, k, v, gate = self.heads(part, first)
            keys.extend(O.four_bits(k, self.cfg["key_scale"]))
            values.extend(O.four_bits(v, self.cfg["value_scale"]))
            K, V = np.array(keys), np.array(values)
            o = np.zeros((n, self.H, self.d))
            for h in range(self.H):
                g = h // (self.H // self.G)
                s_ = q[:, h] @ K[:, g].T * float(np.float32(self.cfg["scale"]))
                s_[np.arange(len(K))[None] > first + np.arange(n)[:, None]] = -np.inf
                w = np.exp(s_ - s_.max(axis=1, keepdims=True))
                o[:, h] = w @ V[:, g] / w.sum(axis=1, keepdims=True)
            o = o.reshape(n, -1)
            outs.append(o if gate is None else o * O.sigmoid(gate))
        return np.concatenate(outs)


class Decay(Rotated):
    """Linear attention with decay."""

    def __init__(self, torch, lib, cfg, precision, slots=3, capacity=2000, eps=1e-3, norm=True, rates=None, **kw):
        super().__init__(torch, lib, cfg, precision, slots, capacity, eps, **kw)
        rng = np.random.default_rng(11)
        self.rates = (-np.exp2(-1 - 9 * rng.random(self.H)) if rates is None else np.asarray(rates)).astype(np.float32)
        self.norm = (1 + 0.2 * rng.standard_normal(self.H * self.d)).astype(np.float32) if norm else None
        self.m = self.capi.DecayMixer(*self.views, self.rotation, self.b.f32(self.rates), self.b.f32(self.norm) if norm else None, self.H, self.d, int(self.gated),
                                      cfg["scale"])
        self.states = torch.zeros((slots, self.H, self.d, self.d), device="cuda")
        self.memory = {}

    def forward(self, route, slots, proj, check_rc=0, advance=True, into=None, pd=None):
        torch, n_seq = self.torch, len(slots)
        n = len(proj) // n_seq
        out = torch.zeros((n_seq * n, self.H * self.d), device="cuda", dtype=self.dtype)
        size = self.lib.tbl_decay_workspace_bytes(C.byref(self.m), self.precision, route, n_seq, n)
        ws = self.space(max(size, 256))
        pd = self.device(proj) if pd is None else pd
        into = self.states if into is None else into
        rc = self.lib.tbl_decay_forward(C.byref(self.m), self.precision, route, self.eps, pd.data_ptr(), self.states.data_ptr(), into.data_ptr(), self.b.i32(slots),
                                        self.positions.data_ptr(), n_seq, n, out.data_ptr(), ws.data_ptr(), size, stream(torch))
        assert rc == check_rc
        if rc == 0 and advance:
            self.positions[slots] += n
        return f64(out)

    def oracle(self, slots, proj):
        """Token by token, [value][key]."""
        n, outs = len(proj) // len(slots), []
        for i, s in enumerate(slots):
            part = proj[i * n:(i + 1) * n]
            m = self.memory.setdefault(s, {"at": 0, "S": np.zeros((self.H, self.d, self.d))})
            q, k, v, gate = self.heads(part, m["at"])
            keep, o = np.exp(self.rates.astype(np.float64)), np.zeros((n, self.H, self.d))
            for t in range(n):
                m["S"] = keep[:, None, None] * m["S"] + v[t][:, :, None] * k[t][:, None, :]
                o[t] = float(np.float32(self.cfg["scale"])) * np.einsum("hvk,hk->hv", m["S"], q[t])
            m["at"] += n
            if self.norm is not None:
                o = O.rms_norm(o, self.norm.reshape(self.H, self.d), self.eps)
            o = o.reshape(n, -1)
            outs.append(o if gate is None else o * O.sigmoid(gate))
        return np.concatenate(outs)
