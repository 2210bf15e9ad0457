"""Linear attention in 64 bits from its definition, a batch of it on the device, and how far a result may be off.

With fade = exp(g) and, beside the state S, its absolute twin A (A = fade A + |k| |v|), what a state's rounding in 32 bits can add up to is
  E = fade E + 2^-22 A      a step's product, sum and factor (2^-24 each, the exponential 2^-23)
and, where factors over several tokens are exponentials of sums of g, the rounding of their arguments
  B = fade (B + |g| A)      sum over tokens of weight * |argument|, times 2^-22 (argument and its product with log2 e).
  A itself               weighted values as operands: two fp16 parts (2^-11 of what 2^-11 leaves: 2^-22 A), three bf16 parts (2^-24 A);
                         a chunk's products are added up by four matrix instructions a part, each with up to two roundings of 2^-24 of the sum:
                         8 x 2 of 2^-24 A for fp16, 12 x 2 for bf16 (E counts them token by token, too few where a token fades at once)
A state may be off by E + 2^-22 B + OPERAND A.  Outputs: scale |q|^T (E + 2^-22 B + 2^-15 A), the last for operands of 16 bits in two parts
(2^-16 each for states and weights) and for the sums over channels (2^-24 each of 128), and half a step of the output."""
import ctypes as C

import torch

from plain_kv import HALF_STEP, HALF_TINY
from oracle import DT_BF16, DT_F16

OPERAND = {DT_F16: 2.0 ** -22 + 16 * 2.0 ** -24, DT_BF16: 2.0 ** -24 + 24 * 2.0 ** -24}
TYPES = {DT_F16: torch.float16, DT_BF16: torch.bfloat16}


class Case:
    """lens: tokens of each request.  decay: None, "head", "token", or a function (tokens, heads) -> tensor of log decays."""

    def __init__(self, lens, dt, k_heads=2, v_heads=4, dk=128, dv=128, decay="token", seed=1, slots=None, state_in="own", state_out="next", kept=None,
                 has_initial=None, mask=None, pads=(0, 0, 0, 0, 0), unit=True, value_scale=1.0, state_scale=0.3):
        import gpu_harness as G

        gen = torch.Generator(device=G.DEV)
        gen.manual_seed(seed)
        self.lens, self.dt, self.hk, self.hv, self.dk, self.dv = list(lens), dt, k_heads, v_heads, dk, dv
        r, n = len(lens), sum(lens)
        self.n, self.scale = n, dk ** -0.5
        rnd = lambda *s: torch.randn(s, generator=gen, device=G.DEV)  # noqa: E731
        norm = (lambda x: x / x.norm(dim=-1, keepdim=True)) if unit else (lambda x: x)

        def rows(x, pad):  # [tokens, row + pad], NaN in the gaps and in two rows behind the last
            y = torch.full((n + 2, x[0].numel() + pad if n else x.shape[1] * x.shape[2] + pad), float("nan"), device=G.DEV, dtype=TYPES[dt])
            y[:n, :x.shape[1] * x.shape[2]] = x.reshape(n, -1).to(TYPES[dt])
            return y

        self.q = rows(norm(rnd(n, k_heads, dk)), pads[0])
        self.k = rows(norm(rnd(n, k_heads, dk)), pads[1])
        self.v = rows(rnd(n, v_heads, dv) * value_scale, pads[2])
        self.out_pad = pads[3]
        if decay is None:
            self.g, self.g_stride = None, 0
        elif decay == "head":
            self.g, self.g_stride = -(2.0 ** (-8.0 * torch.arange(1, v_heads + 1, device=G.DEV).float() / v_heads))[None].contiguous(), 0
        else:
            if decay == "token":
                g = -torch.nn.functional.softplus(rnd(n, v_heads) + torch.linspace(-5, 1, v_heads, device=G.DEV))
            else:
                g = decay(n, v_heads).to(G.DEV).float()
            self.g = torch.full((n + 2, v_heads + pads[4]), float("nan"), device=G.DEV)
            self.g[:n, :v_heads] = g
            self.g_stride = v_heads + pads[4]
        self.num_slots = slots or 2 * r
        self.states = rnd(self.num_slots, v_heads, dk, dv) * state_scale
        i32 = lambda x: None if x is None else torch.tensor(x, dtype=torch.int32, device=G.DEV)  # noqa: E731
        self.in_list = list(range(r)) if state_in == "own" else state_in
        self.out_list = list(range(r, 2 * r)) if state_out == "next" else state_out
        self.kept_list, self.has_list, self.mask_list = kept, has_initial, mask
        starts = [0]
        for x in lens:
            starts.append(starts[-1] + x)
        self.starts = starts
        self.qsl = i32(starts)
        self.state_in, self.state_out, self.kept, self.has = i32(self.in_list), i32(self.out_list), i32(kept), i32(has_initial)
        self.mask = None if mask is None else torch.tensor(mask, dtype=torch.uint8, device=G.DEV)

    def fresh(self):
        """Output and states to be written: rows with a pattern, a copy of the states."""
        import gpu_harness as G

        out = torch.full((self.n + 2, self.hv * self.dv + self.out_pad), 77.0, device=G.DEV, dtype=TYPES[self.dt])
        return out, self.states.clone()

    def structs(self, states, max_q_len=None, total=None):
        import gpu_harness as G
        from warp34_amd import ffi

        at = lambda t: None if t is None else t.data_ptr()  # noqa: E731
        layout = ffi.Warp34LinearStateLayout(states.data_ptr(), 4 * states[0].numel(), self.hk, self.hv, self.dk, self.dv)
        batch = ffi.Warp34LinearBatch(at(self.qsl), at(self.state_in), at(self.has), at(self.state_out), at(self.kept), at(self.mask), len(self.lens),
                                      self.n if total is None else total, max(self.lens) if max_q_len is None else max_q_len, self.scale,
                                      self.q.stride(0), self.k.stride(0), self.v.stride(0), self.hv * self.dv + self.out_pad, self.g_stride, 0)
        return layout, batch

    def call(self, scratch="queried", max_q_len=None, with_out=True, into=None, stream=None, total=None):
        """(out [n, hv, dv], states), both as the device left them; checks what must not have been touched."""
        import gpu_harness as G
        from warp34_amd import ffi

        out, states = into or self.fresh()
        layout, batch = self.structs(states, max_q_len, total)
        lib = G.lib()
        need = lib.warp34_linear_attention_scratch_bytes(C.byref(layout), len(self.lens), batch.total_tokens, batch.max_q_len)
        size = need if scratch == "queried" else scratch
        work = torch.full((size + 64,), 0xA5, dtype=torch.uint8, device=G.DEV)
        torch.cuda.synchronize()
        ex = ffi.Warp34Exec(stream or torch.cuda.current_stream().cuda_stream, work.data_ptr() if size else 0, size, 0)
        fn = lib.warp34_linear_attention_f16 if self.dt == DT_F16 else lib.warp34_linear_attention_bf16
        rc = fn(C.byref(ex), C.byref(layout), C.byref(batch), G.ptr(self.q), G.ptr(self.k), G.ptr(self.v), G.ptr(self.g), G.ptr(out) if with_out else None)
        torch.cuda.synchronize()
        assert rc == 0
        assert bool((work[size:] == 0xA5).all()), "bytes behind the scratch"
        if into is None:
            assert bool((out[self.n:] == 77.0).all()) and bool((out[:, self.hv * self.dv:] == 77.0).all()), "rows or gaps of no request"
        return out[:self.n, :self.hv * self.dv].reshape(self.n, self.hv, self.dv), states

    def want(self):
        """(out, its bound, states, their bound, which rows and slots are written), 64 bits."""
        import gpu_harness as G

        f = dict(dtype=torch.float64, device=G.DEV)
        n, hv, group = self.n, self.hv, self.hv // self.hk
        heads = lambda x, h, d: x[:n, :h * d].double().reshape(n, h, d).repeat_interleave(hv // h, 1)  # noqa: E731
        q, k, v = heads(self.q, self.hk, self.dk), heads(self.k, self.hk, self.dk), heads(self.v, hv, self.dv)
        out, bound = torch.full((n, hv, self.dv), 77.0, **f), torch.zeros((n, hv, self.dv), **f)
        states, s_bound = self.states.double(), torch.zeros(self.states.shape, **f)
        for r, length in enumerate(self.lens):
            if self.mask_list is not None and not self.mask_list[r]:
                continue
            slot = -1 if self.in_list is None or (self.has_list is not None and not self.has_list[r]) else self.in_list[r]
            s = self.states[slot].double() if slot >= 0 else torch.zeros((hv, self.dk, self.dv), **f)
            a, b, e = s.abs(), torch.zeros_like(s), torch.zeros_like(s)
            kept = length if self.kept_list is None else min(max(self.kept_list[r], 0), length)
            for t in range(length + 1):
                if t == kept and self.out_list is not None and self.out_list[r] >= 0:
                    states[self.out_list[r]] = s
                    s_bound[self.out_list[r]] = e + 2.0 ** -22 * b + (OPERAND[self.dt] * a if t else 0)
                if t == length:
                    break
                row = self.starts[r] + t
                if self.g is None:
                    g = torch.zeros((hv, 1, 1), **f)
                else:
                    g = self.g[row if self.g_stride else 0, :hv].double()[:, None, None]
                fade = torch.exp(g)
                kv = k[row][:, :, None] * v[row][:, None, :]
                b = fade * (b + torch.where(fade > 0, -g, 0.0) * a)
                s, a = fade * s + kv, fade * a + kv.abs()
                e = fade * e + 2.0 ** -22 * a
                o = (q[row][:, :, None] * s).sum(1) * self.scale
                out[row] = o
                bound[row] = (q[row].abs()[:, :, None] * (e + 2.0 ** -22 * b + 2.0 ** -15 * a)).sum(1) * self.scale
                bound[row] += HALF_STEP[self.dt] * (o.abs() + bound[row]) + HALF_TINY[self.dt]
        return out, bound, states, s_bound

    def check(self, got, with_out=True, want=None):
        out, bound, states, s_bound = want or self.want()
        if with_out:
            off = (got[0].double() - out).abs() - bound
            assert not bool(torch.isnan(off).any()) and float(off.max() if off.numel() else 0) <= 0, "outputs: %g over the bound" % float(off.max())
        off = (got[1].double() - states).abs() - s_bound
        assert not bool(torch.isnan(off).any()) and float(off.max()) <= 0, "states: %g over the bound" % float(off.max())
