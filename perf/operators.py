"""Cases and plain forms of the operators around the 8-bit paged KV cache.

Operators (each named by a case's "op"):

  rope     rotary positions of the q and k rows of a batch: interleaved or half
           layout, part of the head, scaled for long contexts, forward and
           adjoint (the gradient)
  append   rotate k, quantise k and v to 8 bits with a scale for each block of
           16 tokens and KV head, store them in the pages of their sequences
  decode   one token a sequence: append it, then attend the sequence's rows
  attend   several tokens a sequence: causal attention over cached rows
  fork     share a sequence's pages with others and let each grow by a token
           (the shared last page is copied on write)
  compact  move the pages in use to the lowest page numbers

The cache.  codes [page][layer][kv head][K, V][64 rows][head_dim] in 8 bits
(int8 or e4m3), scales [page][layer][kv head][K, V][4 blocks of 16 rows] FP32;
a value is code * scale.  table [slot][max_pages] holds the pages of each
sequence slot (-1: none), lens [slot] its rows, refs [page] the number of
sequences that hold a page.
"""
import math

import torch

own = False

PAGE, BLOCK = 64, 16
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
LAYOUTS = ("llama", "qwen")            # pairs (2i, 2i+1); pairs (i, i + dim/2)
SCALINGS = ("none", "linear", "yarn", "llama3")


# ------------------------------------------------------------------ cases
def _rope_case(rows, heads, kv_heads, head_dim, dim, layout, scaling, dtype, adjoint, far, **kw):
    return dict(kw, op="rope", rows=rows, heads=heads, kv_heads=kv_heads, head_dim=head_dim, dim=dim,
                layout=layout, scaling=scaling, dtype=dtype, adjoint=adjoint, far=far)


def _kv_case(op, seqs, tokens, length, heads, kv_heads, head_dim, fmt, dtype, ragged, layout="llama", **kw):
    return dict(kw, op=op, seqs=seqs, tokens=tokens, length=length, heads=heads, kv_heads=kv_heads,
                head_dim=head_dim, fmt=fmt, dtype=dtype, ragged=ragged, layout=layout)


def _page_case(op, layers, kv_heads, head_dim, seqs, length, fmt="int8", **kw):
    return dict(kw, op=op, layers=layers, kv_heads=kv_heads, head_dim=head_dim, seqs=seqs, length=length, fmt=fmt)


def listed():
    return [
        # one decode step's q and k rows of 64 sequences, 32/4 heads of 64: a launch, little else
        _rope_case(64, 32, 4, 64, 64, "llama", "none", "float32", False, 4096, name="rope decode 64"),
        # the gradient through the rotation of 8192 training rows, half of a head of 128, long-context scaling
        _rope_case(8192, 32, 8, 128, 64, "qwen", "yarn", "bfloat16", True, 131072, name="rope gradient 8192"),
        # the new rows of a decode step of 64 sequences, into blocks that hold earlier rows
        _kv_case("append", 64, 1, 2048, 4, 4, 64, "int8", "float32", True, name="append decode 64"),
        # ragged prompts of up to 4096 tokens of a prefill batch
        _kv_case("append", 8, 4096, 4096, 8, 8, 128, "e4m3", "bfloat16", True, "qwen", name="append prompts 8x4096"),
        # the smallest call: one sequence, a short context
        _kv_case("decode", 1, 1, 256, 32, 4, 64, "int8", "float32", False, name="decode 1x256"),
        # batched decode, 64 sequences of 2048 rows
        _kv_case("decode", 64, 1, 2048, 32, 4, 64, "int8", "float32", False, name="decode 64x2048"),
        # one long context, split over the whole GPU
        _kv_case("decode", 1, 1, 32768, 32, 8, 64, "e4m3", "bfloat16", False, name="decode 1x32768"),
        # ragged lengths up to 8192 at head_dim 128
        _kv_case("decode", 32, 1, 8192, 32, 8, 128, "int8", "bfloat16", True, "qwen", name="decode ragged 32x8192"),
        # causal prefill of a 2048-token prompt
        _kv_case("attend", 1, 2048, 2048, 32, 4, 64, "int8", "float32", False, name="attend prefill 2048"),
        # ragged chunks of up to 1024 tokens behind contexts of up to 8192 rows
        _kv_case("attend", 4, 1024, 8192, 32, 8, 128, "e4m3", "bfloat16", True, "qwen", name="attend chunks 4x1024"),
        # 63 continuations of one prompt, 22 layers: the shared last page becomes 63 pages
        _page_case("fork", 22, 4, 64, 64, 1000, name="fork 63"),
        # every second sequence has ended: the pages in use move down
        _page_case("compact", 22, 4, 64, 48, 1300, name="compact 48"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("rope", "append", "decode", "decode", "attend", "attend", "fork", "compact"))
    head_dim = rng.choice((64, 128))
    kv_heads = rng.choice((1, 2, 4, 8))
    heads = kv_heads * rng.choice((1, 2, 3, 4, 5, 6, 7, 8))
    dtype = rng.choice(tuple(DTYPES))
    fmt = rng.choice(("int8", "e4m3"))
    layout = rng.choice(LAYOUTS)
    if op == "rope":
        return _rope_case(_log(rng, 1, 8192), min(heads, 32), kv_heads, head_dim, 2 * rng.randint(4, head_dim // 2),
                          layout, rng.choice(SCALINGS), dtype, rng.random() < 0.5, _log(rng, 512, 1 << 20))
    if op == "append":
        tokens = rng.choice((1, _log(rng, 2, 4096)))
        return _kv_case("append", max(1, min(_log(rng, 1, 128), 24576 // tokens)), tokens,
                        tokens + rng.choice((0, _log(rng, 1, 4096))), kv_heads, kv_heads, head_dim, fmt, dtype,
                        True, layout)
    if op == "decode":
        length = _log(rng, 1, 65536)
        return _kv_case("decode", max(1, min(_log(rng, 1, 128), 163840 // (length * kv_heads * head_dim // 1024 + 1))),
                        1, length, heads, kv_heads, head_dim, fmt, dtype, rng.random() < 0.7, layout)
    if op == "attend":
        tokens = _log(rng, 2, 2048)
        heads = min(heads, 32)
        room = (1 << 29) // (tokens * heads)
        length = tokens + rng.choice((0, min(_log(rng, 1, 8192), max(1, room - tokens))))
        return _kv_case("attend", max(1, min(_log(rng, 1, 16), room // length)), tokens, length, heads, kv_heads,
                        head_dim, fmt, dtype, rng.random() < 0.7, layout)
    layers = _log(rng, 1, 22)
    return _page_case(op, layers, rng.choice((1, 2, 4)), 64, _log(rng, 2, 48), _log(rng, 1, 1300), fmt)


def work(case):
    """Bytes and operations that one pass cannot do without; ragged sizes by
    their mean."""
    if case["op"] == "rope":
        n = case["rows"] * (case["heads"] + case["kv_heads"]) * case["head_dim"]
        e = DTYPES[case["dtype"]].itemsize
        return {"bytes": 2 * n * e + 4 * case["rows"], "flops": 3 * n * case["dim"] // case["head_dim"]}
    hk, hd = case["kv_heads"], case["head_dim"]
    if case["op"] in ("fork", "compact"):
        page = case["layers"] * hk * 2 * (PAGE * hd + 4 * PAGE // BLOCK)
        n_seqs, pages = case["seqs"], -(-case["length"] // PAGE)
        tables = 4 * n_seqs * pages
        if case["op"] == "fork":
            copies = n_seqs - 1 if case["length"] % PAGE else 0
        else:
            copies = _mean_moves(n_seqs, pages)
        return {"bytes": 2 * copies * page + 2 * tables, "flops": 0}
    e = DTYPES[case["dtype"]].itemsize
    sizes = _sizes(case)
    tok, rows = sum(n for n, _ in sizes), sum(m for _, m in sizes)
    row_bytes = 2 * hk * hd + 2 * hk * 4 / BLOCK
    if case["op"] == "append":  # k and v in, codes out, and the same rows read back in 16 bits
        back = sum(min(m, max(n, BLOCK)) for n, m in sizes)
        return {"bytes": 2 * tok * hk * hd * e + (tok + back) * row_bytes + 2 * back * hk * hd * 2,
                "flops": 8 * tok * hk * hd}
    q = 2 * tok * case["heads"] * hd * e
    pairs = sum(n * (m - n) + n * (n + 1) // 2 for n, m in sizes)
    extra = 2 * tok * hk * hd * e if case["op"] == "decode" else 0
    return {"bytes": rows * row_bytes + q + extra, "flops": 4 * pairs * case["heads"] * hd}


def _mean_moves(seqs, pages):
    """Pages that move when every second of `seqs` sequences of `pages`
    pages, spread at random, has ended: the used ones in the upper half."""
    used = pages * ((seqs + 1) // 2)
    return used * (seqs * pages - used) // (seqs * pages)


# ----------------------------------------------------------------- inputs
def _sizes(case):
    """(new tokens, rows in the cache with them) of each sequence: whole, or
    spread evenly from a part of the size up to all of it."""
    n, tokens, length = case["seqs"], case["tokens"], case["length"]
    if not case["ragged"] or n == 1:
        return [(tokens, length)] * n
    got = []
    for i in range(n):
        t = max(1, tokens - (i * 7 % n) * tokens // (2 * n))
        got.append((t, max(t, length - (i * 5 % n) * length // (n + n // 4 + 1))))
    return got


def _gen(seed, k=0):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 16 + k)
    return g


def _int(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _rope_params(case):
    """Base and scaling of the case's rotation: (base, scaling, factor, original length, low, high)."""
    scaling = case.get("scaling", "none")
    return {"none": (10000.0, scaling, 1.0, 0, 0.0, 0.0), "linear": (10000.0, scaling, 4.0, 0, 0.0, 0.0),
            "yarn": (500000.0, scaling, 16.0, 8192, 1.0, 32.0),
            "llama3": (500000.0, scaling, 8.0, 8192, 1.0, 4.0)}[scaling]


def _frequencies(dim, base, scaling, factor, orig, low, high):
    """Radians a position of each rotated pair (64 bits) and the factor on
    cosine and sine."""
    i = torch.arange(dim // 2, dtype=torch.float64)
    f = base ** (-2 * i / dim)
    if scaling == "linear":
        return f / factor, 1.0
    if scaling == "yarn":
        bound = [dim * math.log(orig / (turns * 2 * math.pi)) / (2 * math.log(base)) for turns in (high, low)]
        lo, hi = max(math.floor(bound[0]), 0), min(math.ceil(bound[1]), dim - 1)
        ramp = ((i - lo) / max(hi - lo, 0.001)).clamp(0, 1)
        return f / factor * ramp + f * (1 - ramp), 0.1 * math.log(factor) + 1.0
    if scaling == "llama3":
        turns = orig * f / (2 * math.pi)
        smooth = ((turns - low) / (high - low)).clamp(0, 1)
        return f * ((1 - smooth) / factor + smooth), 1.0
    return f, 1.0


def _own_rope(case, dim):
    import picolm_b200 as pb
    base, scaling, factor, orig, low, high = _rope_params(case)
    kind = {"none": pb.PL_ROPE_SCALE_NONE, "linear": pb.PL_ROPE_SCALE_LINEAR, "yarn": pb.PL_ROPE_SCALE_YARN,
            "llama3": pb.PL_ROPE_SCALE_LLAMA3}[scaling]
    layout = pb.PL_ROPE_LLAMA if case["layout"] == "llama" else pb.PL_ROPE_QWEN
    return pb.Rope(case["head_dim"], layout, dim=dim, base=base, scaling=kind, factor=factor, orig_len=orig,
                   low=low, high=high)


def _quantise_pool(shape, fmt, gen):
    """Codes and scales of N(0, 1) rows: shape [pages][layers][heads][2][64][head_dim]."""
    codes = torch.empty(shape, dtype=torch.int8 if fmt == "int8" else torch.float8_e4m3fn, device="cuda")
    scales = torch.empty(shape[:4] + (PAGE // BLOCK,), device="cuda")
    top = 127.0 if fmt == "int8" else 448.0
    for at in range(0, shape[0], 512):
        n = min(512, shape[0] - at)
        x = torch.randn((n,) + shape[1:4] + (PAGE // BLOCK, BLOCK * shape[5]), device="cuda", generator=gen)
        s = x.abs().amax(-1) / top
        x = (x / s[..., None]).clamp(-top, top)
        codes[at:at + n] = (x.round() if fmt == "int8" else x).to(codes.dtype).view((n,) + shape[1:])
        scales[at:at + n] = s
    return codes, scales


def _cache(case, layers, lens, max_pages, spare, gen):
    """A cache whose sequences lie in pages spread over the pool."""
    used = [-(-m // PAGE) for m in lens]
    n_pages = sum(used) + spare
    order = torch.randperm(n_pages, device="cuda", generator=gen).int()
    held = _int(used)
    col = torch.arange(max_pages, device="cuda")[None]
    mine = col < held[:, None]
    table = torch.full((len(lens), max_pages), -1, dtype=torch.int32, device="cuda")
    table[mine] = order[:sum(used)]
    refs = torch.zeros(n_pages, dtype=torch.int32, device="cuda")
    refs[order[:sum(used)].long()] = 1
    codes, scales = _quantise_pool((n_pages, layers, case["kv_heads"], 2, PAGE, case["head_dim"]), case["fmt"], gen)
    return dict(codes=codes, scales=scales, table=table, lens=_int(lens), refs=refs)


def _own_cache(case, s, layers):
    import picolm_b200 as pb
    fmt = pb.PL_KV8_INT8 if case["fmt"] == "int8" else pb.PL_KV8_E4M3
    heads = case.get("heads", case["kv_heads"])
    rope = _own_rope(case, case["head_dim"]) if "layout" in case else None
    geometry = dict(n_layers=layers, n_heads=heads, n_kv_heads=case["kv_heads"], head_dim=case["head_dim"],
                    n_pages=s["refs"].numel(), n_seqs=s["lens"].numel(), max_pages=s["table"].shape[1], fmt=fmt)
    s["work"] = torch.zeros(pb.kv8_work_bytes(**geometry), dtype=torch.uint8, device="cuda")
    return pb.Kv8Cache(**geometry, rope=rope, codes=s["codes"].data_ptr(), scales=s["scales"].data_ptr(),
                       table=s["table"].data_ptr(), lens=s["lens"].data_ptr(), refs=s["refs"].data_ptr(),
                       work=s["work"].data_ptr(), work_bytes=s["work"].numel())


LAYERS, LAYER = 2, 1  # of the attention cases: the second of two layers


def prepare(case, seed):
    gen = _gen(seed)
    if case["op"] == "rope":
        h, hk, hd, n = case["heads"], case["kv_heads"], case["head_dim"], case["rows"]
        # q and k are parts of the rows of a fused projection, padded by a
        # head; decode rows sit at positions of their own, a prompt's follow
        # one another
        rows = torch.randn(n, (h + 2 * hk + 1) * hd, device="cuda", generator=gen).to(DTYPES[case["dtype"]])
        if n <= 128:
            pos = torch.randint(0, case["far"], (n,), device="cuda", generator=gen).int()
        else:
            first = int(torch.randint(0, max(1, case["far"] - n), (1,), device="cuda", generator=gen))
            pos = torch.arange(first, first + n, device="cuda").int()
        freq, factor = _frequencies(case["dim"], *_rope_params(case))
        s = dict(case=case, rows=rows, q=rows[:, :h * hd], k=rows[:, h * hd:(h + hk) * hd], pos=pos,
                 freq=freq.cuda(), factor=factor, q_out=torch.empty(n, h * hd, dtype=rows.dtype, device="cuda"),
                 k_out=torch.empty(n, hk * hd, dtype=rows.dtype, device="cuda"))
        if own:
            s["rope"] = _own_rope(case, case["dim"])
        return s
    if case["op"] in ("fork", "compact"):
        pages, n = -(-case["length"] // PAGE), case["seqs"]
        if case["op"] == "fork":  # slot 0 holds the prompt, the others take it over
            lens = [case["length"]] + [0] * (n - 1)
            s = _cache(case, case["layers"], lens, pages + 1, n + pages + 16, gen)
            s["src"], s["dst"] = _int([0] * (n - 1)), _int(list(range(1, n)))
            s["grown"] = _int([case["length"] + 1] * (n - 1))
        else:
            s = _cache(case, case["layers"], [case["length"]] * n, pages, 16, gen)
            ended = torch.arange(1, n, 2, device="cuda")
            s["refs"][s["table"][ended].long().flatten()] = 0
            s["table"][ended] = -1
            s["lens"][ended] = 0
            # the books as they are before the pass
            s["before"] = [s[x].clone() for x in ("table", "refs")]
        s["case"] = case
        if own:
            s["cache"] = _own_cache(case, s, case["layers"])
        return s
    sizes = _sizes(case)
    tok = [n for n, _ in sizes]
    start = [0]
    for n in tok:
        start.append(start[-1] + n)
    lens = [m for _, m in sizes]
    s = _cache(case, LAYERS, lens, -(-max(lens) // PAGE) + 1, 8, gen)
    h, hk, hd, total = case["heads"], case["kv_heads"], case["head_dim"], start[-1]
    dt = DTYPES[case["dtype"]]
    rows = torch.randn(total, (h + 2 * hk + 1) * hd, device="cuda", generator=gen).to(dt)
    # the batch takes the slots in an order of its own
    order = torch.randperm(len(lens), device="cuda", generator=gen).int()
    s["lens"] = torch.empty_like(s["lens"]).scatter_(0, order.long(), s["lens"])
    s["table"] = torch.empty_like(s["table"]).index_copy_(0, order.long(), s["table"])
    freq, factor = _frequencies(hd, *_rope_params(case))
    s.update(case=case, rows=rows, q=rows[:, :h * hd], k=rows[:, h * hd:(h + hk) * hd],
             v=rows[:, (h + hk) * hd:(h + 2 * hk) * hd], seqs=order, start=_int(start), n=len(lens), total=total, max_tok=max(tok), freq=freq.cuda(),
             factor=factor, max_len=max(lens), out=torch.zeros(total, h * hd, dtype=dt, device="cuda"))
    if case["op"] == "append":
        # read back: the new rows, and the block before them that they joined
        back = [min(m, max(n, BLOCK)) for n, m in sizes]
        first = [0]
        for n in back:
            first.append(first[-1] + n)
        s.update(row0=_int([m - b for (_, m), b in zip(sizes, back)]), back=_int(first), n_back=first[-1],
                 max_back=max(back))
        s.update(k_back=torch.empty(first[-1], hk * hd, dtype=torch.bfloat16, device="cuda"),
                 v_back=torch.empty(first[-1], hk * hd, dtype=torch.bfloat16, device="cuda"))
    if own:
        s["cache"] = _own_cache(case, s, LAYERS)
    return s


# ----------------------------------------------------------------- passes
def run(s):
    return (_run_own if own else _run_plain)(s)


def _run_own(s):
    import picolm_b200 as pb
    case = s["case"]
    op, stream = case["op"], torch.cuda.current_stream().cuda_stream
    if op == "fork":
        c, n = s["cache"], case["seqs"] - 1
        c.fork_dev(n, s["src"].data_ptr(), s["dst"].data_ptr(), stream)
        c.resize_dev(n, s["dst"].data_ptr(), s["grown"].data_ptr(), stream)
        return s["table"], s["lens"], s["refs"], s["codes"], s["scales"]
    if op == "compact":
        s["table"].copy_(s["before"][0])
        s["refs"].copy_(s["before"][1])
        s["cache"].compact_dev(stream)
        return s["table"], s["refs"], s["codes"], s["scales"]
    dtype = {"float32": pb.PL_F32, "bfloat16": pb.PL_BF16, "float16": pb.PL_F16}[case["dtype"]]
    width = s["rows"].stride(0)
    if op == "rope":
        h, hk, hd = case["heads"], case["kv_heads"], case["head_dim"]
        s["rope"].rows_dev(dtype, case["rows"], s["pos"].data_ptr(), h, s["q"].data_ptr(), width,
                           s["q_out"].data_ptr(), h * hd, hk, s["k"].data_ptr(), width, s["k_out"].data_ptr(),
                           hk * hd, case["adjoint"], stream)
        return s["q_out"], s["k_out"]
    c, seqs, start = s["cache"], s["seqs"].data_ptr(), s["start"].data_ptr()
    if op == "append":
        c.append_dev(LAYER, s["n"], seqs, start, s["total"], s["max_tok"], dtype, s["k"].data_ptr(), width,
                     s["v"].data_ptr(), width, stream)
        d = s["k_back"].stride(0)
        c.read_dev(LAYER, s["n"], seqs, s["row0"].data_ptr(), s["back"].data_ptr(), s["n_back"], s["max_back"],
                   pb.PL_BF16, s["k_back"].data_ptr(), d, s["v_back"].data_ptr(), d, stream)
        return s["k_back"], s["v_back"]
    d = s["out"].stride(0)
    if op == "decode":
        c.decode_dev(LAYER, s["n"], seqs, dtype, s["q"].data_ptr(), width, s["k"].data_ptr(), width,
                     s["v"].data_ptr(), width, s["out"].data_ptr(), d, stream)
        return s["out"], s["scales"]
    c.attend_dev(LAYER, s["n"], seqs, start, s["total"], s["max_tok"], dtype, s["q"].data_ptr(), width,
                 s["out"].data_ptr(), d, stream)
    return s["out"]


def _run_plain(s):
    case = s["case"]
    op = case["op"]
    if op == "rope":
        got = []
        for x, n, out in ((s["q"], case["heads"], s["q_out"]), (s["k"], case["kv_heads"], s["k_out"])):
            y = _rotate(x.float().reshape(-1, n, case["head_dim"]), s["pos"], s["freq"], s["factor"], case["layout"],
                        case["adjoint"])
            got.append(out.copy_(y.flatten(1)))
        return got[0], got[1]
    if op == "fork":
        _plain_fork(s)
        _plain_grow(s)
        return s["table"], s["lens"], s["refs"], s["codes"], s["scales"]
    if op == "compact":
        s["table"].copy_(s["before"][0])
        s["refs"].copy_(s["before"][1])
        _plain_compact(s)
        return s["table"], s["refs"], s["codes"], s["scales"]
    if op == "append":
        _plain_append(s)
        return _plain_read(s)
    if op == "decode":
        _plain_append(s)
        return _plain_attend(s), s["scales"]
    return _plain_attend(s)


def _rotate(x, pos, freq, factor, layout, adjoint=False):
    """x [rows][heads][head_dim] in 32 bits; angles in 64."""
    dim = 2 * freq.numel()
    angle = pos.double()[:, None] * freq
    c, sn = (angle.cos() * factor).float()[:, None], (angle.sin() * factor).float()[:, None]
    sn = -sn if adjoint else sn
    y = x.clone()
    a, b = (slice(0, dim, 2), slice(1, dim, 2)) if layout == "llama" else (slice(0, dim // 2), slice(dim // 2, dim))
    y[..., a] = x[..., a] * c - x[..., b] * sn
    y[..., b] = x[..., a] * sn + x[..., b] * c
    return y


def _plain_append(s):
    case = s["case"]
    hk, hd, dev = case["kv_heads"], case["head_dim"], "cuda"
    top = 127.0 if case["fmt"] == "int8" else 448.0
    start, seqs = s["start"].long(), s["seqs"].long()
    lens = s["lens"][seqs].long()
    row0 = lens - (start[1:] - start[:-1])
    n_blocks = (s["max_tok"] + BLOCK - 2) // BLOCK + 1
    rows = (row0 // BLOCK)[:, None, None] * BLOCK + torch.arange(n_blocks * BLOCK, device=dev).view(n_blocks, BLOCK)
    new = (rows >= row0[:, None, None]) & (rows < lens[:, None, None])
    old = rows < row0[:, None, None]
    some = new.any(-1)
    at = torch.where(new, start[:-1, None, None] + rows - row0[:, None, None], 0)
    page = s["table"][seqs[:, None], (rows[..., 0] // PAGE).clamp(max=s["table"].shape[1] - 1)].long().clamp(min=0)
    sub = rows[..., 0] % PAGE // BLOCK
    # which sequence and position each token has, for its rotation
    tok = torch.arange(s["total"], device=dev)
    of = torch.searchsorted(start[1:].contiguous(), tok, right=True)
    pos = row0[of] + tok - start[of]
    k = _rotate(s["k"].float().reshape(-1, hk, hd), pos, s["freq"], s["factor"], case["layout"])
    both = torch.stack((k, s["v"].float().reshape(-1, hk, hd)), 2)             # [token][head][2][hd]
    # [seq][block][row][head][2][hd]
    x = torch.where(new[..., None, None, None], both[at], 0.0)
    have = s["codes"].view(-1, LAYERS, hk, 2, PAGE // BLOCK, BLOCK, hd)
    was = have[page, LAYER, :, :, sub].float().permute(0, 1, 4, 2, 3, 5)
    s_old = s["scales"][page, LAYER, :, :, sub]                                 # [seq][block][head][2]
    s_new = x.abs().amax((2, 5)) / top
    s_new = torch.where(old.any(-1)[..., None, None], torch.maximum(s_old, s_new), s_new)
    safe = torch.where(s_new > 0, s_new, 1.0)[:, :, None, :, :, None]
    ratio = torch.where(s_new > 0, s_old / torch.where(s_new > 0, s_new, 1.0), 1.0)[:, :, None, :, :, None]
    code = torch.where(old[..., None, None, None], was * ratio, x / safe).clamp(-top, top)
    code = (code.round() if case["fmt"] == "int8" else code).to(s["codes"].dtype)
    i, b, r = (some[..., None] & (old | new)).nonzero(as_tuple=True)
    flat = s["codes"].view(-1, LAYERS, hk, 2, PAGE, hd)
    flat.view(torch.int8)[page[i, b], LAYER, :, :, rows[i, b, r] % PAGE] = code.view(torch.int8)[i, b, r]
    i, b = some.nonzero(as_tuple=True)
    s["scales"][page[i, b], LAYER, :, :, sub[i, b]] = s_new[i, b]


def _values(s, rows_to):
    """K and V of the batch's sequences, [seq][head][row][hd] in 32 bits, of
    the rows below rows_to."""
    hk, hd = s["case"]["kv_heads"], s["case"]["head_dim"]
    pages = -(-rows_to // PAGE)
    page = s["table"][s["seqs"].long(), :pages].long().clamp(min=0)
    x = s["codes"][page, LAYER].float().view(s["n"], pages, hk, 2, PAGE // BLOCK, BLOCK, hd)
    x = x * s["scales"][page, LAYER][..., None, None]
    x = x.view(s["n"], pages, hk, 2, PAGE, hd).permute(3, 0, 2, 1, 4, 5).reshape(2, s["n"], hk, pages * PAGE, hd)
    return x[0], x[1]


def _plain_read(s):
    hk, hd = s["case"]["kv_heads"], s["case"]["head_dim"]
    back, row = s["back"].long(), torch.arange(s["n_back"], device="cuda")
    of = torch.searchsorted(back[1:].contiguous(), row, right=True)
    at = s["row0"].long()[of] + row - back[of]
    page = s["table"][s["seqs"].long()[of], at // PAGE].long()
    codes = s["codes"][page, LAYER, :, :, at % PAGE].float()
    x = codes * s["scales"][page, LAYER, :, :, at % PAGE // BLOCK][..., None]
    s["k_back"].copy_(x[:, :, 0].reshape(-1, hk * hd))
    s["v_back"].copy_(x[:, :, 1].reshape(-1, hk * hd))
    return s["k_back"], s["v_back"]


def _plain_attend(s):
    case = s["case"]
    h, hk, hd, n, dev = case["heads"], case["kv_heads"], case["head_dim"], s["n"], "cuda"
    start, t = s["start"].long(), s["max_tok"]
    lens = s["lens"][s["seqs"].long()].long()
    count = start[1:] - start[:-1]
    j = torch.arange(t, device=dev)
    real = j < count[:, None]
    at = torch.where(real, start[:-1, None] + j, 0)
    pos = (lens - count)[:, None] + j                                        # [seq][token]
    k, v = _values(s, s["max_len"])
    col = torch.arange(k.shape[2], device=dev)
    v = torch.where((col < lens[:, None])[:, None, :, None], v, 0.0)
    q = _rotate(s["q"].float().reshape(-1, h, hd)[at].view(n * t, h, hd), pos.flatten(), s["freq"], s["factor"],
                case["layout"])
    q = q.view(n, t, hk, h // hk, hd).permute(0, 2, 3, 1, 4).reshape(n, hk, h // hk * t, hd)
    seen = col <= pos.repeat(1, h // hk)[:, :, None]                         # [seq][group, token][row]
    p = (q @ k.transpose(2, 3)) / math.sqrt(hd)
    p = p.masked_fill_(~seen[:, None], -math.inf)
    top = p.amax(-1, keepdim=True)
    p = p.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    o = (p @ v) / p.sum(-1, keepdim=True).clamp(min=1e-30)
    o = o.view(n, hk, h // hk, t, hd).permute(0, 3, 1, 2, 4).reshape(n, t, h * hd)
    s["out"][at[real]] = o[real].to(s["out"].dtype)
    return s["out"]


def _plain_fork(s):
    """Slots dst give up their pages and share those of src."""
    src, dst, refs = s["src"].long(), s["dst"].long(), s["refs"]
    for slots, by in ((dst, -1), (src, 1)):
        page = s["table"][slots].long()
        refs.index_add_(0, page.clamp(min=0).flatten(), torch.where(page >= 0, by, 0).int().flatten())
    s["table"][dst] = s["table"][src]
    s["lens"][dst] = s["lens"][src]


def _copy_pages(s, src, dst):
    s["codes"].view(torch.int8)[dst] = s["codes"].view(torch.int8)[src]
    s["scales"][dst] = s["scales"][src]


def _plain_grow(s):
    """Slots dst grow to s["grown"] rows (by less than a page): a new page
    where the last one is full, a copy of the last one where it is shared
    (the last sharer of the list keeps it if nobody else holds it).  New
    pages are the lowest free ones, in the order of the list."""
    dst, refs, table = s["dst"].long(), s["refs"], s["table"]
    old, new = s["lens"][dst].long(), s["grown"].long()
    last = (new - 1) // PAGE
    fresh = old % PAGE == 0
    page = table[dst, last].long()
    same = (page[:, None] == page) & ~fresh[:, None] & ~fresh
    rank = same.tril(-1).sum(1)
    copy = ~fresh & (refs[page.clamp(min=0)] - rank > 1)
    need = fresh | copy
    free = (refs == 0).nonzero()[:, 0]
    got = torch.where(need, free[(need.cumsum(0) - 1).clamp(min=0)], page)
    _copy_pages(s, page[copy], got[copy])
    refs.index_add_(0, page[copy], torch.full_like(page[copy], -1, dtype=torch.int32))
    refs[got[need]] = 1
    table[dst, last] = got.int()
    s["lens"][dst] = s["grown"]


def _plain_compact(s):
    refs, table = s["refs"], s["table"]
    used = refs > 0
    top = used.sum()
    index = torch.arange(refs.numel(), device="cuda")
    src = (used & (index >= top)).nonzero()[:, 0]
    dst = (~used & (index < top)).nonzero()[:, 0]
    _copy_pages(s, src, dst)
    to = index.clone()
    to[src] = dst
    table.copy_(torch.where(table >= 0, to[table.long().clamp(min=0)].int(), table))
    refs[dst] = refs[src]
    refs[src] = 0


# ------------------------------------------------------------------ 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op in ("fork", "compact"):
        return None  # pages are moved, nothing is computed
    base, scaling, factor, orig, low, high = _rope_params(case)
    dim = case.get("dim", case["head_dim"])
    freq, gain = [], 1.0
    for i in range(dim // 2):
        w = math.pow(base, -2.0 * i / dim)
        if scaling == "linear":
            w /= factor
        elif scaling == "llama3":
            wave = 2 * math.pi / w
            if wave > orig / low:
                w /= factor
            elif wave >= orig / high:
                mix = (orig / wave - low) / (high - low)
                w = (1 - mix) * w / factor + mix * w
        elif scaling == "yarn":
            first = max(math.floor(dim * math.log(orig / (high * 2 * math.pi)) / (2 * math.log(base))), 0)
            last = min(math.ceil(dim * math.log(orig / (low * 2 * math.pi)) / (2 * math.log(base))), dim - 1)
            part = min(max((i - first) / (last - first if last > first else 0.001), 0.0), 1.0)
            w = w / factor * part + w * (1 - part)
            gain = 0.1 * math.log(factor) + 1
        freq.append(w)
    freq = torch.tensor(freq, dtype=torch.float64, device="cuda")

    def turn(x, pos, back=False):  # [..., rows, heads, hd], as complex numbers
        by = torch.polar(torch.full_like(pos.double()[:, None] * freq, gain), pos.double()[:, None] * freq)
        by = (by.conj() if back else by)[:, None]
        x = x.double()
        if case["layout"] == "llama":
            z = torch.view_as_complex(x[..., :dim].reshape(x.shape[:-1] + (dim // 2, 2)).contiguous()) * by
            return torch.cat((torch.view_as_real(z).flatten(-2), x[..., dim:]), -1)
        z = torch.complex(x[..., :dim // 2], x[..., dim // 2:dim]) * by
        return torch.cat((z.real, z.imag, x[..., dim:]), -1)

    if op == "rope":
        return tuple(turn(x.unflatten(1, (-1, case["head_dim"])), s["pos"], case["adjoint"]).flatten(1)
                     for x in (s["q"], s["k"]))
    hk, hd, group = case["kv_heads"], case["head_dim"], case["heads"] // case["kv_heads"]
    if op == "attend" and work(case)["flops"] > 4e12:
        return None
    start, seqs, lens = s["start"].tolist(), s["seqs"].tolist(), s["lens"].tolist()
    top = 127.0 if case["fmt"] == "int8" else 448.0
    outs, backs, scales = [], [], s["scales"].double()
    for i, slot in enumerate(seqs):
        m, n = lens[slot], start[i + 1] - start[i]
        first = m - n
        pages = s["table"][slot, :-(-m // PAGE)].long()
        code = s["codes"][pages, LAYER].double()                      # [page][head][2][64][hd]
        scale = s["scales"][pages, LAYER].double()                    # [page][head][2][4]
        pos = torch.arange(first, m, device="cuda")
        if op != "attend":
            k = turn(s["k"][start[i]:start[i + 1]].unflatten(1, (hk, hd)), pos)
            v = s["v"][start[i]:start[i + 1]].double().unflatten(1, (hk, hd))
            code = code.permute(1, 2, 0, 3, 4).flatten(2, 3).contiguous()  # [head][2][row][hd]
            scale = scale.permute(1, 2, 0, 3).flatten(2, 3).contiguous()   # [head][2][block]
            x = torch.zeros_like(code)
            x[:, 0, first:m], x[:, 1, first:m] = k.transpose(0, 1), v.transpose(0, 1)
            blk = slice(first // BLOCK, (m - 1) // BLOCK + 1)
            in_new = torch.zeros(code.shape[2], dtype=torch.bool, device="cuda")
            in_new[first:m] = True
            largest = torch.where(in_new[:, None], x.abs(), 0).unflatten(2, (-1, BLOCK)).amax((3, 4))
            # the scale is held in 32 bits: that is its definition
            want = (largest / top).float().double()
            if first % BLOCK:
                want[..., first // BLOCK] = torch.maximum(want[..., first // BLOCK], scale[..., first // BLOCK])
            to = scale.clone()
            to[..., blk] = want[..., blk]
            scales[pages, LAYER] = to.unflatten(2, (-1, PAGE // BLOCK)).permute(2, 0, 1, 3)
            each = to.repeat_interleave(BLOCK, 2)[..., None]
            kept = code * torch.where(each > 0, scale.repeat_interleave(BLOCK, 2)[..., None] / each, 1.0)
            y = torch.where(in_new[:, None], torch.where(each > 0, x / each, 0.0), kept).clamp(-top, top)
            y = y.round() if case["fmt"] == "int8" else _to_e4m3(y)
            touched = torch.zeros_like(in_new)
            touched[blk.start * BLOCK:m] = True
            value = torch.where(touched[:, None], y, code) * each
        else:
            value = (code.unflatten(3, (4, BLOCK)) * scale[..., None, None]).flatten(3, 4)
            value = value.permute(1, 2, 0, 3, 4).flatten(2, 3)
        if op == "append":
            at = slice(m - min(m, max(n, BLOCK)), m)
            backs.append(value[:, :, at].permute(2, 1, 0, 3).flatten(2))   # [row][2][heads * hd]
            continue
        q = turn(s["q"][start[i]:start[i + 1]].unflatten(1, (-1, hd)), pos)
        got = torch.empty(n, hk * group, hd, dtype=torch.float64, device="cuda")
        step = max(1, (1 << 27) // (m * group))
        for g in range(hk):
            for a in range(0, n, step):
                z = torch.einsum("tgd,rd->tgr", q[a:a + step, g * group:(g + 1) * group], value[g, 0, :m]) / hd ** 0.5
                hide = torch.arange(m, device="cuda") > pos[a:a + step, None]
                z = torch.softmax(z.masked_fill(hide[:, None], -math.inf), -1)
                got[a:a + step, g * group:(g + 1) * group] = torch.einsum("tgr,rd->tgd", z, value[g, 1, :m])
        outs.append(got.flatten(1))
    if op == "append":
        both = torch.cat(backs)
        return both[:, 0].contiguous(), both[:, 1].contiguous()
    return (torch.cat(outs), scales) if op == "decode" else torch.cat(outs)


def _to_e4m3(x):
    """Nearest value with 3 bits behind the leading one and exponents from -6
    (halves to even), from 64 bits."""
    e = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6)))
    e = torch.where(x.abs() >= torch.exp2(e + 1), e + 1, torch.where(x.abs() < torch.exp2(e), e - 1, e)).clamp(min=-6)
    step = torch.exp2(e - 3)
    return torch.round(x / step) * step
