"""Plain 64-bit forms of the rotary operator and of the 8-bit paged cache,
and a cache in torch memory, for the tests of pl_rope_* and pl_kv8_*."""
import math

import torch

import picolm_b200 as pb

PAGE, BLOCK = pb.PL_KV8_PAGE, pb.PL_KV8_BLOCK
TORCH = {pb.PL_F32: torch.float32, pb.PL_F16: torch.float16, pb.PL_BF16: torch.bfloat16}
DTYPES = tuple(TORCH)
TOP = {pb.PL_KV8_INT8: 127.0, pb.PL_KV8_E4M3: 448.0}


def frequencies(dim, base=10000.0, scaling=pb.PL_ROPE_SCALE_NONE, factor=1.0, orig_len=0, low=1.0, high=4.0):
    """(radians a position of each pair, gain) of a pl_rope, from its definition."""
    out, gain = [], 1.0
    for i in range(dim // 2):
        f = base ** (-2.0 * i / dim)
        turns = orig_len * f / (2 * math.pi)
        if scaling == pb.PL_ROPE_SCALE_LINEAR:
            f = f / factor
        elif scaling == pb.PL_ROPE_SCALE_LLAMA3:
            keep = min(max((turns - low) / (high - low), 0.0), 1.0)
            f = keep * f + (1 - keep) * f / factor
        elif scaling == pb.PL_ROPE_SCALE_YARN:
            def at(t):
                return dim * math.log(orig_len / (t * 2 * math.pi)) / (2 * math.log(base))
            lo, hi = max(math.floor(at(high)), 0), min(math.ceil(at(low)), dim - 1)
            part = min(max((i - lo) / max(hi - lo, 0.001), 0.0), 1.0)
            f = part * f / factor + (1 - part) * f
            gain = 0.1 * math.log(factor) + 1
        out.append(f)
    return torch.tensor(out, dtype=torch.float64), gain


def rotate(x, pos, freq, gain, layout, adjoint=False):
    """x [rows][heads][head_dim] in 64 bits, pos [rows]."""
    x = x.double()
    dim = 2 * len(freq)
    angle = pos.double()[:, None] * freq.to(x.device)
    c, s = gain * angle.cos()[:, None], gain * angle.sin()[:, None] * (-1 if adjoint else 1)
    y = x.clone()
    a, b = ((slice(0, dim, 2), slice(1, dim, 2)) if layout == pb.PL_ROPE_LLAMA
            else (slice(0, dim // 2), slice(dim // 2, dim)))
    y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., a] * s + x[..., b] * c
    return y


class Cache:
    """A Kv8Cache over torch tensors."""

    def __init__(self, heads, kv_heads, head_dim=64, fmt=pb.PL_KV8_INT8, n_pages=32, n_seqs=4, max_pages=8,
                 layers=1, layout=pb.PL_ROPE_LLAMA, rope_dim=None, **rope_kw):
        self.heads, self.kv_heads, self.head_dim, self.fmt, self.layers = heads, kv_heads, head_dim, fmt, layers
        self.layout, self.dim = layout, head_dim if rope_dim is None else rope_dim
        self.freq, self.gain = frequencies(self.dim, **rope_kw)
        shape = (n_pages, layers, kv_heads, 2, PAGE, head_dim)
        # memory that nothing wrote: garbage codes and NaN scales
        self.codes = torch.randint(-128, 128, shape, device="cuda").to(torch.int8)
        self.scales = torch.full(shape[:4] + (PAGE // BLOCK,), math.nan, device="cuda")
        self.table = torch.full((n_seqs, max_pages), -1, dtype=torch.int32, device="cuda")
        self.lens = torch.zeros(n_seqs, dtype=torch.int32, device="cuda")
        self.refs = torch.zeros(n_pages, dtype=torch.int32, device="cuda")
        geometry = dict(n_layers=layers, n_heads=heads, n_kv_heads=kv_heads, head_dim=head_dim, n_pages=n_pages,
                        n_seqs=n_seqs, max_pages=max_pages, fmt=fmt)
        self.work = torch.zeros(pb.kv8_work_bytes(**geometry), dtype=torch.uint8, device="cuda")
        rope = pb.Rope(head_dim, layout, dim=self.dim, **rope_kw)
        self.c = pb.Kv8Cache(**geometry, rope=rope, codes=self.codes.data_ptr(), scales=self.scales.data_ptr(),
                             table=self.table.data_ptr(), lens=self.lens.data_ptr(), refs=self.refs.data_ptr(),
                             work=self.work.data_ptr(), work_bytes=self.work.numel())

    # calls with torch arguments -----------------------------------------
    def resize(self, seqs, lens=None, want=pb.PL_OK):
        s, n = i32(seqs), None if lens is None else i32(lens)
        self.c.resize_dev(len(seqs), s.data_ptr(), None if n is None else n.data_ptr(), stream())
        assert self.c.status(stream()) == want

    def fork(self, src, dst, want=pb.PL_OK):
        a, b = i32(src), i32(dst)
        self.c.fork_dev(len(src), a.data_ptr(), b.data_ptr(), stream())
        assert self.c.status(stream()) == want

    def compact(self):
        self.c.compact_dev(stream())
        assert self.c.status(stream()) == pb.PL_OK

    def append(self, seqs, counts, k, v, dtype, layer=0):
        s, st = i32(seqs), i32(starts(counts))
        self.c.append_dev(layer, len(seqs), s.data_ptr(), st.data_ptr(), sum(counts), max(counts), dtype,
                          k.data_ptr(), k.stride(0), v.data_ptr(), v.stride(0), stream())
        assert self.c.status(stream()) == pb.PL_OK

    def attend(self, seqs, counts, q, out, dtype, layer=0, max_tok=None):
        s, st = i32(seqs), i32(starts(counts))
        self.c.attend_dev(layer, len(seqs), s.data_ptr(), st.data_ptr(), sum(counts), max_tok or max(counts), dtype,
                          q.data_ptr(), q.stride(0), out.data_ptr(), out.stride(0), stream())
        assert self.c.status(stream()) == pb.PL_OK
        return out

    def decode(self, seqs, q, k, v, out, dtype, layer=0):
        s = i32(seqs)
        self.c.decode_dev(layer, len(seqs), s.data_ptr(), dtype, q.data_ptr(), q.stride(0), k.data_ptr(),
                          k.stride(0), v.data_ptr(), v.stride(0), out.data_ptr(), out.stride(0), stream())
        assert self.c.status(stream()) == pb.PL_OK
        return out

    # what the memory holds ----------------------------------------------
    def values(self, slot, rows, layer=0):
        """K and V of rows [0, rows) of a slot in 64 bits: [2][rows][kv head][head_dim]."""
        pages = self.table[slot, :-(-rows // PAGE)].long()
        code = self.codes[pages, layer]
        code = (code if self.fmt == pb.PL_KV8_INT8 else code.view(torch.float8_e4m3fn).float()).double()
        scale = self.scales[pages, layer].double().repeat_interleave(BLOCK, -1)
        x = (code * scale[..., None]).permute(2, 0, 3, 1, 4).reshape(2, -1, self.kv_heads, self.head_dim)
        return x[:, :rows]

    def fill(self, seqs, lens, gen, layer=0, scale=1.0):
        """Grow slots to `lens` rows of random codes, written directly."""
        self.resize(seqs, lens)
        for slot, m in zip(seqs, lens):
            for p in self.table[slot, :-(-m // PAGE)].tolist():
                x = torch.randn(self.codes.shape[2:], device="cuda", generator=gen) * scale
                blk = x.view(self.kv_heads, 2, PAGE // BLOCK, -1)
                s = blk.abs().amax(-1) / TOP[self.fmt]
                y = (blk / s[..., None]).clamp(-TOP[self.fmt], TOP[self.fmt]).view(x.shape)
                self.codes[p, layer] = (y.round().to(torch.int8) if self.fmt == pb.PL_KV8_INT8
                                        else y.to(torch.float8_e4m3fn).view(torch.int8))
                self.scales[p, layer] = s
            self.spoil(slot, m, layer)

    def spoil(self, slot, rows, layer=0):
        """What lies behind a slot's last row: NaN codes (e4m3) or -128, and
        NaN scales of blocks without a row."""
        if rows % PAGE == 0:
            return
        p = int(self.table[slot, rows // PAGE])
        self.codes[p, layer, :, :, rows % PAGE:] = 127 if self.fmt == pb.PL_KV8_E4M3 else -128
        self.scales[p, layer, :, :, -(-(rows % PAGE) // BLOCK):] = math.nan

    def reference(self, seqs, counts, q, layer=0):
        """Attention of q in 64 bits over what the memory holds, the largest
        sum |q k| / sqrt(hd) of a score and the largest |v|."""
        outs, most, vmax, t = [], 0.0, 0.0, 0
        group = self.heads // self.kv_heads
        for slot, n in zip(seqs, counts):
            m = int(self.lens[slot])
            pos = torch.arange(m - n, m, device="cuda")
            qr = rotate(q[t:t + n].double().view(n, self.heads, self.head_dim), pos, self.freq, self.gain, self.layout)
            t += n
            k, v = self.values(slot, m, layer)
            k, v = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
            s = torch.einsum("thd,rhd->htr", qr, k) / math.sqrt(self.head_dim)
            hide = torch.arange(m, device="cuda") > pos[:, None]
            p = torch.exp(s.masked_fill(hide, -math.inf) - s.masked_fill(hide, -math.inf).amax(-1, keepdim=True)
                          if m else s)
            p = torch.nan_to_num(p / p.sum(-1, keepdim=True)) if m else p
            p[:, pos < 0] = 0
            outs.append(torch.einsum("htr,rhd->thd", p, v).flatten(1))
            if m and n:
                most = max(most, float(torch.einsum("thd,rhd->htr", qr.abs(), k.abs()).max()) / math.sqrt(self.head_dim))
                vmax = max(vmax, float(v.abs().max()))
        return torch.cat(outs), most, vmax


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def starts(counts):
    s = [0]
    for n in counts:
        s.append(s[-1] + n)
    return s


def stream():
    return torch.cuda.current_stream().cuda_stream


def generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def randn(gen, *shape, dtype=torch.float32):
    return torch.randn(*shape, device="cuda", generator=gen).to(dtype)


def attention_bound(dtype, head_dim, rows, most, vmax, want):
    """How far an attention output may be from 64 bits.

    With u = 2^-24 (FP32) and S = max sum |q k| / sqrt(hd): the rotation of q
    is off by at most 8u relative (reduced angle, cosine, two products and a
    sum), q as two FP16 parts by 2^-22 = 4u, the dot product by (hd + 2) u
    per term, the scales by 2u, so a score by (hd + 16) u S, and 2^x by 2^-22
    and the argument's own rounding: a weight is off by w = ((hd + 16) S + 2 S
    + 8) u relative.  Numerator and denominator each sum `rows` weights (rows
    * u relative), and the weight takes two FP16 parts (4u): out <= vmax (2 w
    + 2 rows u + 8u).  Sixteen-bit activations may take q and the weight as one FP16
    value: S 2^-11 on a score and 2^-11 on a weight more; and the output is
    rounded once, by half a step."""
    u = 2.0 ** -24
    w = ((head_dim + 18) * most + 8) * u
    bound = vmax * (2 * w + (2 * rows + 8) * u)
    if dtype != pb.PL_F32:
        bound = bound + vmax * 2 * (most + 1) * 2.0 ** -11 + want.abs() * torch.finfo(TORCH[dtype]).eps / 2
        bound = bound + torch.finfo(TORCH[dtype]).tiny
    return bound
