"""RMSNorm + quantization and the linear on E4M3 codes with float32 scales per
128, against the formulas in 64 bits.

Tolerances.  Norm: a row's sum of squares is added in float32, at most 64
terms one after the other and the rest in a tree, rsqrt and the products add a
few roundings: the relative error of a quotient is below 1e-5, so a code must
be the E4M3 rounding of a value within 1e-5 of the exact quotient, and a scale
within 1e-5 of the exact one.  Linear: one bf16 rounding (2^-8 relative) and
float32 sums of 128 products and of the blocks, which the tensor cores may
truncate instead of rounding: (128 + blocks) * 2^-22 of the sum of magnitudes."""

import pytest
import torch

from _e4m3_ref import E4M3, check_close, check_codes

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _setup():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA GPU")
    import voyager_b200  # noqa: F401

    yield


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _exact_norm(x, weight, eps, residual):
    h = x.double() + (residual.double() if residual is not None else 0)
    y = h * (h.square().mean(-1, keepdim=True) + eps).rsqrt() * weight.double() if weight is not None else h
    C = y.shape[-1]
    b = torch.nn.functional.pad(y, (0, -C % 128)).reshape(y.shape[:-1] + (-1, 128))
    s = b.abs().amax(-1) / 448
    s = torch.where(s == 0, 1.0, s)
    return (b / s[..., None]).reshape(y.shape[:-1] + (-1,))[..., :C], s


def _check_norm(x, weight, eps=1e-5, residual=None):
    from voyager_b200 import fp8block

    if weight is None:
        (codes, scale), hidden = fp8block.quantize(x), None
    else:
        codes, scale, hidden = fp8block.rmsnorm_quantize(x, weight, eps, residual)
    q, s = _exact_norm(x, weight, eps, residual)
    assert codes.dtype == E4M3 and codes.shape == x.shape and scale.shape == s.shape
    check_close(scale, s, s * 1e-5)
    check_codes(codes, q, 1e-5)
    if residual is None:
        assert hidden is None
    else:
        assert torch.equal(hidden, (x.float() + residual.float()).to(x.dtype))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("R,C", [(1, 1), (1, 127), (3, 128), (2, 129), (5, 4096), (1, 11008), (7, 1000),
                                 (300, 264), (2, 16384), (2, 32768), (2, 32776), (9, 5003), (3, 40001)])
def test_norm(R, C, dtype):
    g = _gen(R * 100003 + C)
    x, r = (torch.randn(R, C, generator=g, device="cuda").to(dtype) for _ in range(2))
    w = (1 + 0.2 * torch.randn(C, generator=g, device="cuda")).to(dtype)
    _check_norm(x, w)
    _check_norm(x, w, residual=r)
    _check_norm(x, None)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("R,C", [(7000, 264), (9001, 250), (6000, 633), (3000, 1630), (1500, 4104), (700, 11007)])
def test_norm_many_rows(R, C, dtype):
    """More rows than CTAs: each takes several, with the next one in flight."""
    g = _gen(R + C)
    x, r = (torch.randn(R, C, generator=g, device="cuda").to(dtype) for _ in range(2))
    w = (1 + 0.2 * torch.randn(C, generator=g, device="cuda")).to(dtype)
    _check_norm(x, w)
    _check_norm(x, w, residual=r)
    _check_norm(x, None)


@pytest.mark.parametrize("C", [384, 401])
def test_norm_strides_and_shapes(C):
    """Leading dims, row strides beyond the row, starts off 16 bytes, a
    residual of other strides, a strided weight, no rows."""
    g = _gen(C)
    big = torch.randn(2, 5, C + 21, generator=g, device="cuda").bfloat16()
    w = torch.randn(2 * C, generator=g, device="cuda").bfloat16()[::2]
    r = torch.randn(C, 2, 5, generator=g, device="cuda").bfloat16().permute(1, 2, 0)
    for x in (big[..., :C], big[..., 3:C + 3], big[..., 8:C + 8]):
        _check_norm(x, w)
        _check_norm(x, w, residual=r)
        _check_norm(x[0], w, residual=r[1])
        _check_norm(x[1, 2], w, residual=r[0, 0])
    from voyager_b200 import fp8block

    codes, scale, hidden = fp8block.rmsnorm_quantize(big[:0, :, :C], w, residual=r[:0])
    assert codes.shape == (0, 5, C) and scale.shape == (0, 5, (C + 127) // 128) and hidden.shape == codes.shape


@pytest.mark.parametrize("C", [1, 128, 300])
def test_norm_overlapping_rows(C):
    """Rows shared by expansion, and windows of one row that overlap."""
    g = _gen(C)
    x = torch.randn(4, 3, C, generator=g, device="cuda").bfloat16()
    w = torch.randn(C, generator=g, device="cuda").bfloat16()
    one = torch.randn(2 * C + 40, generator=g, device="cuda").bfloat16()
    for t in (one[:C].expand(4, 3, C), one.as_strided((4, 3, C), (3, 1, 1)), one[:C].expand(12, C)):
        v = x.reshape(t.shape)
        _check_norm(t, w)
        _check_norm(t, w, residual=v)
        _check_norm(v, w, residual=t)


def test_norm_special_values():
    """All-zero blocks get scale 1; a NaN makes its row's codes NaN (and only
    its row's), without a norm its block's; large and tiny rows stay exact."""
    from voyager_b200 import fp8block

    g = _gen(1)
    x = torch.randn(6, 512, generator=g, device="cuda")
    w = torch.ones(512, device="cuda")
    x[0] = 0
    x[1, 128:256] = 0
    x[2, 300] = float("nan")
    x[3] *= 1e15
    x[4] *= 1e-18
    for t, ww in ((x, w), (x.bfloat16(), w.bfloat16())):
        q, s = _exact_norm(t, ww, 1e-5, None)
        codes, scale, _ = fp8block.rmsnorm_quantize(t, ww, 1e-5)
        assert bool(codes[2].float().isnan().all()) and bool(scale[2].isnan().all())
        keep = [0, 1, 3, 4, 5]
        check_close(scale[keep], s[keep], s[keep] * 1e-5)
        check_codes(codes[keep], q[keep], 1e-5)
        assert float(scale[0, 0]) == 1.0 and float(scale[1, 1]) == 1.0
        codes, scale = fp8block.quantize(t)
        assert bool(codes[2, 256:384].float().isnan().all()) and bool(scale[2, 2].isnan())
        assert not bool(codes[2, :256].float().isnan().any()) and not bool(scale[2, :2].isnan().any())


@pytest.mark.parametrize("C", [1024, 1022, 1021, 40001])
def test_quantize_extremes(C):
    """Blocks whose largest magnitude lies at the ends of float32's range: the
    codes follow the quotient in the reals, the scale is rounded once more
    where it is denormal, a scale that underflows counts as 0 (scale 1), and an
    infinity leaves 0 in the rest of its block."""
    from voyager_b200 import fp8block

    g = _gen(2)
    x = torch.rand(2, C, generator=g, device="cuda") * 2 - 1
    tops = [3.4e38, 1e38, 2.0**-118, 2.0**-119, 2.0**-126, 2.0**-135]
    for b, top in enumerate(tops):
        x[:, b * 128] = 1
        x[:, b * 128:(b + 1) * 128] *= top
    x[0, 6 * 128:7 * 128] *= 2.0**-147
    x[1, 6 * 128 + 5] = -float("inf")
    x[1, 7 * 128 + 5] = float("nan")
    codes, scale = fp8block.quantize(x)
    q, s = _exact_norm(x, None, 0.0, None)
    n = len(tops)
    check_close(scale[:, :n], s[:, :n], s[:, :n] * 1e-5 + 2.0**-149)
    check_codes(codes[:, :n * 128], q[:, :n * 128], 1e-5)
    assert scale[0, 6] == 1 and bool((codes[0, 6 * 128:7 * 128].float() == 0).all())
    c = codes[1, 6 * 128:7 * 128].float()
    assert scale[1, 6] == float("inf") and bool(c[5].isnan()) and bool((torch.cat([c[:5], c[6:]]) == 0).all())
    assert bool(scale[1, 7].isnan()) and bool(codes[1, 7 * 128:8 * 128].float().isnan().all())


def test_quantize_weight():
    from voyager_b200 import fp8block

    w = torch.randn(300, 200, generator=_gen(2), device="cuda") * 0.02
    w[128:256, :128] = 0
    codes, scale = fp8block.quantize_weight(w)
    assert codes.shape == w.shape and codes.is_contiguous() and scale.shape == (3, 2)
    assert float(scale[1, 0]) == 1.0
    s = scale.double().repeat_interleave(128, 0)[:300].repeat_interleave(128, 1)[:, :200]
    check_close(codes.double() * s, w.double(), w.double().abs() * 2.0 ** -4 + s * 2.0 ** -10)


def _linear_case(M, N, K, seed, bias=True, codes=None):
    from voyager_b200 import fp8block

    g = _gen(seed)
    nk = (K + 127) // 128
    a = (torch.randn(M, K, generator=g, device="cuda") * 100).clamp(-448, 448).to(E4M3)
    w = (torch.randn(N, K, generator=g, device="cuda") * 100).clamp(-448, 448).to(E4M3)
    sa = torch.exp2(torch.randn(M, nk, generator=g, device="cuda") * 2 - 6)
    sw = torch.exp2(torch.randn((N + 127) // 128, nk, generator=g, device="cuda") * 2 - 6)
    b = torch.randn(N, generator=g, device="cuda").bfloat16() if bias else None
    out = fp8block.linear(a, sa, w, sw, b)
    assert out.dtype == torch.bfloat16 and out.shape == (M, N)
    fa = a.double() * sa.double().repeat_interleave(128, 1)[:, :K]
    fw = w.double() * sw.double().repeat_interleave(128, 0)[:N].repeat_interleave(128, 1)[:, :K]
    want = fa @ fw.T + (b.double() if bias else 0)
    mag = fa.abs() @ fw.abs().T
    check_close(out, want, want.abs() * 2.0 ** -8 + mag * (128 + nk) * 2.0 ** -22)
    return out


@pytest.mark.parametrize("M", [1, 2, 15, 16, 17, 32, 33, 64, 65, 128, 129, 200, 257, 700])
@pytest.mark.parametrize("N,K", [(1, 16), (128, 128), (130, 144), (1000, 2048), (257, 4112)])
def test_linear(M, N, K):
    _linear_case(M, N, K, M * 31 + N + K, bias=(M + N) % 2 == 0)


@pytest.mark.parametrize("M,N,K", [(1, 12288, 4096), (16, 4096, 11008), (3000, 4099, 512), (4096, 11008, 256),
                                   (64, 22016, 128), (2, 70000, 64), (1, 128, 65536)])
def test_linear_large(M, N, K):
    _linear_case(M, N, K, N)


@pytest.mark.parametrize("M", [3, 16, 30, 64])
@pytest.mark.parametrize("N,K", [(20000, 720), (19001, 5008), (4096, 12304)])
def test_linear_few_tokens_many_tiles(M, N, K):
    """More tiles than SMs and fewer; K beyond one filling of the scales."""
    _linear_case(M, N, K, M + N)


def test_linear_views_and_empty():
    """Leading dims, operands that are not contiguous, no rows."""
    from voyager_b200 import fp8block

    g = _gen(9)
    x = torch.randn(3, 5, 256, generator=g, device="cuda")
    w = torch.randn(96, 256, generator=g, device="cuda")
    c, s = fp8block.quantize(x)
    wc, ws = fp8block.quantize_weight(w)
    want = fp8block.linear(c.reshape(15, 256), s.reshape(15, 2), wc, ws)
    assert torch.equal(fp8block.linear(c, s, wc, ws), want.view(3, 5, 96))
    ct = c.view(torch.uint8).transpose(0, 1).contiguous().transpose(0, 1).view(E4M3)
    st = s.permute(2, 0, 1).contiguous().permute(1, 2, 0)
    wt = wc.view(torch.uint8).T.contiguous().T.view(E4M3)
    assert torch.equal(fp8block.linear(ct, st, wt, ws.T.contiguous().T), want.view(3, 5, 96))
    assert fp8block.linear(c[:0], s[:0], wc, ws).shape == (0, 5, 96)


def test_linear_special_values():
    """A NaN code reaches its row (activation) or column (weight) and no other;
    infinite scales reach theirs."""
    from voyager_b200 import fp8block

    for M in (3, 200):
        a, w = (torch.ones(n, 256, device="cuda").to(E4M3) for n in (M, 300))
        sa, sw = torch.ones(M, 2, device="cuda"), torch.ones(3, 2, device="cuda")
        a.view(torch.uint8)[1, 7] = 0x7F
        w.view(torch.uint8)[290, 200] = 0xFF
        sa[0, 1] = float("inf")
        out = fp8block.linear(a, sa, w, sw)
        want = torch.full((M, 300), 256.0, device="cuda", dtype=torch.bfloat16)
        want[0] = float("inf")
        want[1] = want[:, 290] = float("nan")
        assert torch.equal(out.isnan(), want.isnan())
        assert torch.equal(torch.nan_to_num(out, 7.0), torch.nan_to_num(want, 7.0))


def test_linear_offsets_past_32_bits():
    """More than 2^31 outputs: the last rows are written where they belong."""
    from voyager_b200 import fp8block

    M, N = 131200, 16500
    a = torch.zeros(M, 16, device="cuda").to(E4M3)
    a.view(torch.uint8)[-3:] = 0x38  # 1.0
    w = torch.ones(N, 16, device="cuda").to(E4M3)
    out = fp8block.linear(a, torch.ones(M, 1, device="cuda"), w, torch.ones((N + 127) // 128, 1, device="cuda"))
    assert bool((out[-3:] == 16).all()) and not bool(out[:-3:997].any()) and not bool(out[-9:-3].any())


def test_other_stream_and_graph():
    """The launches are ordered on the current stream and can be captured."""
    from voyager_b200 import fp8block

    g = _gen(4)
    x = torch.randn(40, 1024, generator=g, device="cuda").bfloat16()
    w = torch.ones(1024, device="cuda").bfloat16()
    wc, ws = fp8block.quantize_weight(torch.randn(512, 1024, generator=g, device="cuda"))
    c, s, _ = fp8block.rmsnorm_quantize(x, w)
    want = fp8block.linear(c, s, wc, ws)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        y = x * 1
        c2, s2, _ = fp8block.rmsnorm_quantize(y, w)
        got = fp8block.linear(c2, s2, wc, ws)
    side.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c3, s3, _ = fp8block.rmsnorm_quantize(y, w)
        out = fp8block.linear(c3, s3, wc, ws)
    y.copy_(-x)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, -want)


def test_refusals():
    from voyager_b200 import fp8block

    x = torch.randn(4, 256, device="cuda").bfloat16()
    w = torch.ones(256, device="cuda").bfloat16()
    with pytest.raises(NotImplementedError):
        fp8block.rmsnorm_quantize(x.half(), w.half())
    with pytest.raises(ValueError):
        fp8block.rmsnorm_quantize(x, w.float())
    with pytest.raises(ValueError):
        fp8block.rmsnorm_quantize(x, w[:128])
    with pytest.raises(ValueError):
        fp8block.rmsnorm_quantize(x, w, residual=x[:2])
    with pytest.raises(ValueError):
        fp8block.rmsnorm_quantize(x[:, :0], w[:0])
    c, s = fp8block.quantize(x)
    wc, ws = fp8block.quantize_weight(torch.randn(96, 256, device="cuda"))
    for bad in ((c.float(), s, wc, ws), (c, s.double(), wc, ws)):
        with pytest.raises(NotImplementedError):
            fp8block.linear(*bad)
    for bad in ((c, s[:, :1], wc, ws), (c[:, :128], s, wc, ws), (c, s, wc, ws[:, :1]), (c, s, wc[:0], ws[:0])):
        with pytest.raises(ValueError):
            fp8block.linear(*bad)
    with pytest.raises(ValueError):
        fp8block.linear(c, s, wc, ws, bias=torch.zeros(96, device="cuda"))
    c8, s8 = fp8block.quantize(x[:, :24])
    with pytest.raises(ValueError):
        fp8block.linear(c8, s8, *fp8block.quantize_weight(torch.randn(96, 24, device="cuda")))
