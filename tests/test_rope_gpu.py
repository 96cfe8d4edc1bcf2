"""rope(): rotary positions against the definition in 64 bits.

Tolerance: the rotation is two fp32 products and a sum of inputs that are
exact in fp32, with cosine and sine good to a few fp32 ulps, then one rounding
to the 16-bit type: |error| <= u |y| + 16 * 2^-24 (|x0| + |x1|) amplitude,
u the type's unit roundoff (2^-11 fp16, 2^-8 bf16), plus half of fp16's
smallest step. It was fixed before the first run.
"""

import math

import pytest
import torch

from conftest import requires_gpu

import flashattn_cuda

pytestmark = [pytest.mark.gpu, requires_gpu]

UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def exact(x, positions, freqs, interleaved, inverse=False, amplitude=1.0):
    """64-bit rotation of x (B, H, N, D) and the sum |x0| + |x1| of each
    element's pair (zero where it is copied)."""
    r = 2 * freqs.numel()
    angle = positions.double().reshape(-1, 1, positions.shape[-1], 1) * freqs.double()
    c = angle.cos() * amplitude
    s = angle.sin() * amplitude * (-1.0 if inverse else 1.0)
    y, size = x.double().clone(), torch.zeros(x.shape, dtype=torch.float64, device=x.device)
    first, second = ((slice(0, r, 2), slice(1, r, 2)) if interleaved
                     else (slice(0, r // 2), slice(r // 2, r)))
    x0, x1 = x[..., first].double(), x[..., second].double()
    y[..., first], y[..., second] = x0 * c - x1 * s, x1 * c + x0 * s
    size[..., first] = size[..., second] = (x0.abs() + x1.abs()) * abs(amplitude)
    return y, size


def check(got, x, *args, **kw):
    want, size = exact(x, *args, **kw)
    tol = UNIT[x.dtype] * want.abs() + 16 * 2.0 ** -24 * size + 2.0 ** -25
    r = 2 * args[1].numel()
    assert got.dtype == x.dtype and got.shape == x.shape and got.is_contiguous()
    assert bool(((got.double() - want).abs() <= tol).all())
    assert torch.equal(got[..., r:], x[..., r:])  # copied, bit for bit


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("b,h,h_kv,n,d,rot", [
    (1, 1, 1, 1, 64, 64), (2, 14, 2, 77, 64, 64), (3, 5, 5, 333, 128, 128),
    (2, 32, 8, 1000, 128, 64), (1, 3, 1, 50, 64, 16), (1, 2, 2, 9, 80, 20),
    (2, 3, 1, 700, 96, 34), (1, 2, 1, 5, 7, 6), (1, 1, 1, 3, 1024, 1024),
    (1, 2, 1, 4, 64, 2), (1, 300, 40, 2, 64, 64)])
def test_rope_matches_the_definition(dtype, interleaved, b, h, h_kv, n, d, rot):
    torch.manual_seed(b * n + d)
    q = torch.randn(b, h, n, d, device="cuda").to(dtype)
    k = torch.randn(b, h_kv, n, d, device="cuda").to(dtype)
    freqs, _ = flashattn_cuda.rope_frequencies(rot)
    positions = torch.randint(0, 200000, (b, n), device="cuda", dtype=torch.int32)
    for inverse, amplitude in ((False, 1.0), (True, 1.25)):
        qo, ko = flashattn_cuda.rope(q, k, positions, freqs, interleaved, inverse,
                                     amplitude)
        check(qo, q, positions, freqs, interleaved, inverse=inverse, amplitude=amplitude)
        check(ko, k, positions, freqs, interleaved, inverse=inverse, amplitude=amplitude)


@pytest.mark.parametrize("interleaved", [False, True])
def test_rope_of_views_and_unaligned_rows(interleaved):
    torch.manual_seed(1)
    b, h, h_kv, n, d = 2, 6, 2, 130, 64
    freqs, _ = flashattn_cuda.rope_frequencies(d)
    positions = torch.arange(5, 5 + n, device="cuda", dtype=torch.int32)
    fused = torch.randn(b, n, h + 2 * h_kv, d, device="cuda").half().transpose(1, 2)
    odd = torch.randn(b, h + 1, n, d + 3, device="cuda").half()[:, 1:, :, 1:d + 1]
    shared = torch.randn(1, h, 1, d, device="cuda").half().expand(b, h, n, d)
    for x in (fused[:, :h], odd, shared):
        qo, ko = flashattn_cuda.rope(x, fused[:, h:h + h_kv], positions, freqs, interleaved)
        check(qo, x, positions, freqs, interleaved)
        check(ko, fused[:, h:h + h_kv], positions, freqs, interleaved)
    qo, ko = flashattn_cuda.rope(odd, None, positions, freqs, interleaved)
    assert ko is None
    check(qo, odd, positions, freqs, interleaved)
    pairs = positions.repeat(b * 2, 1)[::2]  # strided rows of positions
    qo, _ = flashattn_cuda.rope(fused[:, :h], None, pairs, freqs, interleaved)
    check(qo, fused[:, :h], pairs, freqs, interleaved)


def test_rope_far_and_negative_positions_keep_their_angle():
    freqs, _ = flashattn_cuda.rope_frequencies(128)
    positions = torch.tensor([0, -1, -70000, 2 ** 24 + 1, 2 ** 31 - 1, -2 ** 31],
                             device="cuda", dtype=torch.int32)
    x = torch.randn(1, 2, 6, 128, device="cuda").half()
    y, _ = flashattn_cuda.rope(x, None, positions, freqs)
    check(y, x, positions, freqs, False)
    assert torch.equal(y[:, :, 0], x[:, :, 0])  # position 0 turns nothing


def test_rope_special_values_stay_in_their_pair():
    freqs, _ = flashattn_cuda.rope_frequencies(64)
    x = torch.randn(1, 1, 2, 64, device="cuda").half()
    x[0, 0, 0, 3] = float("nan")
    x[0, 0, 1, 40] = float("inf")
    y, _ = flashattn_cuda.rope(x, None, torch.tensor([7, 9], device="cuda",
                                                     dtype=torch.int32), freqs)
    bad = (~y.isfinite()).nonzero()[:, 2:].tolist()
    assert bad == [[0, 3], [0, 35], [1, 8], [1, 40]]


def test_rope_empty():
    freqs, _ = flashattn_cuda.rope_frequencies(64)
    q = torch.empty(2, 3, 0, 64, device="cuda").half()
    y, z = flashattn_cuda.rope(q, q, torch.empty(0, device="cuda", dtype=torch.int32), freqs)
    assert y.shape == q.shape and z.shape == q.shape


@pytest.mark.parametrize("interleaved", [False, True])
def test_rope_gradient(interleaved):
    """inverse=True against differences of the forward call: with g and x in
    whole 1/8ths, sum(g * rope(x)) changes by the gradient's element times
    the step, up to the roundings of the forward results that changed."""
    torch.manual_seed(3)
    n, d = 9, 64
    freqs, amplitude = flashattn_cuda.rope_frequencies(32, scaling="yarn", factor=4.0,
                                                       original_length=64)
    positions = torch.arange(100, 100 + n, device="cuda", dtype=torch.int32)
    x = (torch.randint(-16, 17, (1, 2, n, d), device="cuda") / 8).half()
    g = (torch.randint(-16, 17, (1, 2, n, d), device="cuda") / 8).half()

    def forward(v):
        return flashattn_cuda.rope(v, None, positions, freqs, interleaved,
                                   amplitude=amplitude)[0].double()

    grad, _ = flashattn_cuda.rope(g, None, positions, freqs, interleaved, inverse=True,
                                  amplitude=amplitude)
    check(grad, g, positions, freqs, interleaved, inverse=True, amplitude=amplitude)
    step = 1.0
    for e in (0, 5, 16, 21, 31, 40, 63):
        hi, lo = x.clone(), x.clone()
        hi[..., e] += step
        lo[..., e] -= step
        change = ((forward(hi) - forward(lo)) * g.double()).sum(-1) / (2 * step)
        # two changed results a side, each |y| <= 8 rounded by 2^-11 |y|, times |g| <= 2
        assert bool(((change - grad[..., e].double()).abs() <= 4 * 8 * 2.0 ** -11 * 2 / 2
                     + 2.0 ** -9).all())


def test_rope_on_another_stream():
    freqs, _ = flashattn_cuda.rope_frequencies(64)
    positions = torch.arange(2000, device="cuda", dtype=torch.int32)
    s = torch.cuda.Stream()
    x = torch.randn(4, 8, 2000, 64, device="cuda").half()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        x = x * 2
        y, _ = flashattn_cuda.rope(x, None, positions, freqs)
    s.synchronize()
    check(y, x, positions, freqs, False)


def test_rope_refusals():
    freqs, _ = flashattn_cuda.rope_frequencies(64)
    q = torch.randn(1, 2, 8, 64, device="cuda").half()
    p = torch.arange(8, device="cuda", dtype=torch.int32)

    def refuses(match, *args, **kw):
        with pytest.raises(RuntimeError, match=match):
            flashattn_cuda.rope(*args, **kw)

    refuses("CUDA", q.cpu(), None, p, freqs)
    refuses("fp16 or bf16", q.float(), None, p, freqs)
    refuses("4-D", q[0], None, p, freqs)
    refuses("contiguous along head_dim", q.transpose(2, 3), None, p, freqs)
    refuses("same dtype", q, q.bfloat16(), p, freqs)
    refuses("agree on batch", q, q[:, :, :4], p, freqs)
    refuses("float64", q, None, p, freqs.float())
    refuses("one entry per rotated pair", q, None, p, torch.ones(33, device="cuda").double())
    refuses("one entry per rotated pair", q, None, p, torch.ones(0, device="cuda").double())
    refuses("int32", q, None, p.long(), freqs)
    refuses("positions must be", q, None, p[:7], freqs)
    refuses("amplitude", q, None, p, freqs, amplitude=math.inf)
