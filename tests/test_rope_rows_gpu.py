"""pl_rope_rows_dev on the GPU against the rotation in 64 bits."""
import pytest
import torch

import picolm_b200 as pb
from tests.kv8_util import DTYPES, TORCH, frequencies, generator, i32, randn, rotate, stream

pytestmark = pytest.mark.gpu

SCALED = {
    "none": {},
    "linear": dict(scaling=pb.PL_ROPE_SCALE_LINEAR, factor=4.0),
    "yarn": dict(scaling=pb.PL_ROPE_SCALE_YARN, base=500000.0, factor=16.0, orig_len=8192, low=1.0, high=32.0),
    "llama3": dict(scaling=pb.PL_ROPE_SCALE_LLAMA3, base=500000.0, factor=8.0, orig_len=8192, low=1.0, high=4.0),
}


def bound(x, gain, dtype):
    """Two products and a sum in FP32 of cosine and sine rounded to FP32, each
    2^-24: 4 * 2^-24 of |x_a| + |x_b| times the gain; then half a step of the
    type."""
    big = gain * 2 * x.double().abs().amax(-1, keepdim=True)
    return big * 4 * 2.0 ** -24 + (0 if dtype == pb.PL_F32 else big * torch.finfo(TORCH[dtype]).eps / 2)


def run(rope, dtype, pos, q, k, q_out, k_out, h, hk, adjoint=False):
    p = i32(pos)
    rope.rows_dev(dtype, len(pos), p.data_ptr(), h, q.data_ptr(), q.stride(0), q_out.data_ptr(), q_out.stride(0), hk,
                  k.data_ptr(), k.stride(0), k_out.data_ptr(), k_out.stride(0), adjoint, stream())
    torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", [pb.PL_ROPE_LLAMA, pb.PL_ROPE_QWEN])
@pytest.mark.parametrize("head_dim,dim,scaled", [(64, 64, "none"), (128, 128, "llama3"), (128, 64, "yarn"),
                                                 (64, 32, "linear"), (80, 20, "none"), (256, 256, "yarn"), (8, 2, "none"),
                                                 (64, 0, "none"), (96, 90, "linear"), (128, 16, "none")])
@pytest.mark.parametrize("rows,h,hk", [(1, 32, 4), (37, 5, 1)])
def test_rows(dtype, layout, head_dim, dim, scaled, rows, h, hk):
    gen = generator(rows)
    kw = SCALED[scaled]
    rope = pb.Rope(head_dim, layout, dim=dim, **kw)
    freq, gain = frequencies(dim, **kw)
    # fused projection rows, and an output with padding of its own
    wide = randn(gen, rows, (h + 2 * hk) * head_dim, dtype=TORCH[dtype])
    q, k = wide[:, :h * head_dim], wide[:, h * head_dim:(h + hk) * head_dim]
    pos = [(i * 104729 + 7 * rows) % 1000003 for i in range(rows)]
    for adjoint in (False, True):
        qo = torch.full((rows + 1, h * head_dim + 8), 7.0, dtype=TORCH[dtype], device="cuda")
        ko = torch.full((rows + 1, hk * head_dim), 7.0, dtype=TORCH[dtype], device="cuda")
        run(rope, dtype, pos, q, k, qo, ko, h, hk, adjoint)
        for x, y, n in ((q, qo, h), (k, ko, hk)):
            x3 = x.reshape(rows, n, head_dim)
            want = rotate(x3, i32(pos), freq, gain, layout, adjoint)
            got = y[:rows, :n * head_dim].reshape(rows, n, head_dim)
            assert bool(((got.double() - want).abs() <= bound(x3, gain, dtype)).all())
            assert torch.equal(got[..., dim:], x3[..., dim:])
            assert bool((y[rows:] == 7).all()) and bool((y[:, n * head_dim:] == 7).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", [pb.PL_ROPE_LLAMA, pb.PL_ROPE_QWEN])
def test_in_place_unaligned_and_far(dtype, layout):
    gen = generator(3)
    rope = pb.Rope(64, layout, dim=48)
    freq, gain = frequencies(48)
    flat = randn(gen, 9 * 201 + 3, dtype=TORCH[dtype])
    x = torch.as_strided(flat, (9, 192), (201, 1), 3)   # odd strides, rows that start anywhere
    before = x.clone()
    pos = [0, 1, 2 ** 31 - 1, 10 ** 9, 5, 4096, 131071, 7, 3]
    run(rope, dtype, pos, x, x, x, x, 3, 0)
    want = rotate(before.reshape(9, 3, 64), i32(pos), freq, gain, layout)
    # the angle in 64 bits: position times frequency is off by 2^-53 of up to 2^31 radians
    assert bool(((x.reshape(9, 3, 64).double() - want).abs() <=
                 bound(before.reshape(9, 3, 64), gain, dtype) + 16 * 2.0 ** -22).all())


def test_many_rows():
    gen = generator(4)
    rope = pb.Rope(128, pb.PL_ROPE_QWEN)
    freq, gain = frequencies(128)
    q, k = randn(gen, 5001, 4 * 128, dtype=torch.bfloat16), randn(gen, 5001, 128, dtype=torch.bfloat16)
    qo, ko = torch.empty_like(q), torch.empty_like(k)
    run(rope, pb.PL_BF16, list(range(5001)), q, k, qo, ko, 4, 1)
    for x, y, n in ((q, qo, 4), (k, ko, 1)):
        x3 = x.view(5001, n, 128)
        want = rotate(x3, torch.arange(5001, device="cuda"), freq, gain, pb.PL_ROPE_QWEN)
        assert bool(((y.view(5001, n, 128).double() - want).abs() <= bound(x3, gain, pb.PL_BF16)).all())


@pytest.mark.parametrize("layout", [pb.PL_ROPE_LLAMA, pb.PL_ROPE_QWEN])
def test_adjoint_is_the_gradient(layout):
    """<J x, y> = <x, J' y>, and J' y equals the differences of <J x, y>
    along each element: J is linear, so a difference over h = 1 is exact but
    for rounding (the bound of the two sums of 64 products)."""
    gen = generator(5)
    kw = SCALED["yarn"]
    rope = pb.Rope(64, layout, dim=40, **kw)
    x, y = randn(gen, 3, 64), randn(gen, 3, 64)
    jx, jty = torch.empty_like(x), torch.empty_like(y)
    pos = [5, 77777, 9]
    run(rope, pb.PL_F32, pos, x, x, jx, x.clone(), 1, 0)
    run(rope, pb.PL_F32, pos, y, y, jty, y.clone(), 1, 0, adjoint=True)
    slack = 64 * 2.0 ** -22 * 8 * 8
    assert float(((jx.double() * y.double()).sum(1) - (x.double() * jty.double()).sum(1)).abs().max()) <= slack
    for e in range(64):
        x2 = x.clone()
        x2[:, e] += 1
        j2 = torch.empty_like(x)
        run(rope, pb.PL_F32, pos, x2, x2, j2, x.clone(), 1, 0)
        diff = ((j2.double() - jx.double()) * y.double()).sum(1)
        assert float((diff - jty[:, e].double()).abs().max()) <= slack


def test_captured_and_on_another_stream():
    gen = generator(6)
    rope = pb.Rope(64)
    freq, gain = frequencies(64)
    x, out, pos = randn(gen, 4, 256), torch.zeros(4, 256, device="cuda"), i32([1, 2, 3, 4])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rope.rows_dev(pb.PL_F32, 4, pos.data_ptr(), 4, x.data_ptr(), 256, out.data_ptr(), 256, stream=stream())
    x.copy_(randn(gen, 4, 256))
    pos.add_(1000)
    graph.replay()
    torch.cuda.synchronize()
    want = rotate(x.view(4, 4, 64), pos, freq, gain, pb.PL_ROPE_LLAMA)
    assert bool(((out.view(4, 4, 64).double() - want).abs() <= bound(x.view(4, 4, 64), gain, pb.PL_F32)).all())
    del graph
