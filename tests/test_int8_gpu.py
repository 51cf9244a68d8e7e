"""Rows in 8 bits and their product against the formulas in 64 bits.

Codes are compared for equality: with p_i = x_i or s_i w_i exact in 64 bits
and P = max|p|, code_i = rint(127 p_i / P).  A scale is one fp32 rounding
(2^-24) of a quotient held in 64 bits.  The product's sum is exact; it is
rounded to fp32 (2^-24), multiplied by two scales and added to the bias, one
rounding each, and rounded to the output's type (finfo.eps / 2)."""

import pytest
import torch

from coda_gqa_l import Int8Rows, _hip, linear_int8, quantize_rows, rms_norm_int8

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]
WIDTHS = [(1, 1), (3, 7), (2, 64), (5, 127), (70, 128), (6, 129), (4, 1000), (3, 1024), (9, 1025), (2, 2047), (3, 2048),
          (2, 4096), (3, 5000), (2, 8191), (2, 8192), (1, 8200), (2, 16384), (1, 30001), (2, 32768), (300, 96)]


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _rand(g, *shape, dtype=torch.float32, std=1.0):
    return (torch.randn(*shape, generator=g, device=DEV) * std).to(dtype)


def _codes64(p):
    """Codes and largest magnitudes of rows p in 64 bits."""
    top = p.abs().amax(-1, keepdim=True)
    return torch.where(top > 0, torch.round(p * 127.0 / top), 0.0), top


def _check_rows(r, codes, scales):
    """r's codes equal, its scales within one rounding, zeros behind."""
    K = r.cols
    assert r.codes.shape[-1] == -(-K // 128) * 128
    assert torch.equal(r.codes[..., :K].double(), codes)
    assert not r.codes[..., K:].any()
    assert ((r.scales.double() - scales).abs() <= scales * U * 1.0001).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,D", WIDTHS)
def test_quantize_rows(M, D, dtype):
    x = _rand(_gen(M + D), M, D, dtype=dtype, std=3.0)
    r = quantize_rows(x)
    codes, top = _codes64(x.double())
    _check_rows(r, codes, top[:, 0] / 127)
    assert r.shape == x.shape and r.dtype == dtype
    # a value: code times scale in fp32, then rounded to the type
    want = r.codes[:, :D].double() * r.scales.double()[:, None]
    for to in (None, torch.float32):
        got = r.dequantize(to).double()
        assert ((got - want).abs() <= want.abs() * (U + torch.finfo(to or dtype).eps / 2) + 2.0 ** -25).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,D", WIDTHS)
@pytest.mark.parametrize("residual", [True, False])
def test_rms_norm_int8(M, D, dtype, residual):
    g = _gen(7 * M + D)
    x, w = _rand(g, M, D, dtype=dtype, std=0.5), (1 + 0.3 * _rand(g, D)).to(dtype)
    s = x
    if residual:
        res = _rand(g, M, D, dtype=dtype, std=2.0)
        s = (x.float() + res.float()).to(dtype)
        r, out = rms_norm_int8(x, w, 1e-5, residual=res)
        assert torch.equal(out, s)
    else:
        r = rms_norm_int8(x, w, 1e-5)
    codes, top = _codes64(s.double() * w.double())
    rms = torch.sqrt(s.double().pow(2).mean(-1) + float(torch.tensor(1e-5, dtype=torch.float32)))
    _check_rows(r, codes, top[:, 0] / 127 / rms)


def _views(g, kind, dtype, M=6, D=256):
    if kind == "wide rows":
        return _rand(g, M, D + 40, dtype=dtype)[:, :D]
    if kind == "off 16 bytes":
        return _rand(g, M * D + 1, dtype=dtype)[1:].view(M, D)
    if kind == "odd stride":
        return _rand(g, M, D + 3, dtype=dtype)[:, 2:D + 2]
    if kind == "transposed":
        return _rand(g, D, M, dtype=dtype).t()
    if kind == "one row, expanded":
        return _rand(g, 1, D, dtype=dtype).expand(M, D)
    if kind == "four dims":
        return _rand(g, 2, 3, 5, D, dtype=dtype).transpose(0, 2)
    return _rand(g, D, dtype=dtype)  # one dim


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", ["wide rows", "off 16 bytes", "odd stride", "transposed", "one row, expanded",
                                  "four dims", "one dim"])
def test_layouts(kind, dtype):
    """Every layout gives what a dense copy gives."""
    g = _gen(5)
    x, res = _views(g, kind, dtype), _views(g, kind, dtype)
    w = _views(g, "off 16 bytes", dtype, 1)[0]
    a, b = quantize_rows(x), quantize_rows(x.clone(memory_format=torch.contiguous_format))
    assert torch.equal(a.codes, b.codes) and torch.equal(a.scales, b.scales) and a.shape == x.shape
    (a, s), (b, t) = (rms_norm_int8(x, w, residual=res),
                      rms_norm_int8(x.clone(memory_format=torch.contiguous_format), w.clone(),
                                    residual=res.clone(memory_format=torch.contiguous_format)))
    assert torch.equal(a.codes, b.codes) and torch.equal(a.scales, b.scales) and torch.equal(s, t)
    assert a.scales.shape == x.shape[:-1] and s.shape == x.shape


@pytest.mark.parametrize("D", [16, 24, 700, 4096])
@pytest.mark.parametrize("dtype", TYPES)
def test_halves_go_to_even(D, dtype):
    """p / P 127 on a half exactly: P = 254, p odd integers below it."""
    p = torch.arange(D, device=DEV).mul(2).add(1).remainder(254).to(dtype)
    p[::3] *= -1
    p[D // 2] = 254
    r = quantize_rows(p[None])
    assert torch.equal(r.codes[0, :D].double(), torch.round(p.double() / 2))
    w = torch.ones_like(p)
    assert torch.equal(rms_norm_int8(p[None], w).codes, r.codes)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [5, 512, 5000])
def test_rows_that_hold_no_number(D, dtype):
    """Zeros: scale 0.  An infinity or a NaN: scale NaN, codes 0, and nothing
    of it reaches another row."""
    g = _gen(D)
    x = _rand(g, 5, D, dtype=dtype)
    x[1] = 0
    x[2, D // 2], x[3, D - 1] = float("inf"), float("nan")
    w = torch.ones(D, device=DEV, dtype=dtype)
    for r in (quantize_rows(x), rms_norm_int8(x, w), rms_norm_int8(x, w, 0.0, residual=torch.zeros_like(x))[0]):
        assert r.scales[1] == 0 and r.scales[2:4].isnan().all() and not r.codes[1:4].any()
        assert torch.isfinite(r.scales[[0, 4]]).all() and (r.codes[[0, 4]].abs().amax(1) == 127).all()
        y = linear_int8(r, quantize_rows(_rand(g, 9, D, dtype=dtype)))
        assert not y[1].any() and y[2:4].isnan().all() and torch.isfinite(y[[0, 4]]).all()
        v = r.dequantize()
        assert not v[1].any() and v[2:4].isnan().all()
    w[0] = float("nan")
    assert rms_norm_int8(x, w).scales.isnan().all()
    # an overflow of the sum with the residual
    big = torch.full((1, D), torch.finfo(dtype).max, dtype=dtype, device=DEV)
    r, s = rms_norm_int8(big, torch.ones_like(w), residual=big)
    assert s.isinf().all() and r.scales.isnan().all()


@pytest.mark.parametrize("dtype,size", [(torch.float32, 1e30), (torch.float32, 1e-30), (torch.bfloat16, 1e30),
                                        (torch.bfloat16, 1e-30), (torch.float16, 6e4), (torch.float16, 1e-7)])
def test_sizes_beyond_fp32_squares(dtype, size):
    x = (torch.rand(3, 300, generator=_gen(1), device=DEV) * size).to(dtype)
    w = torch.full((300,), 2.0, device=DEV, dtype=dtype)
    r = rms_norm_int8(x, w, 0.0)
    codes, top = _codes64(x.double() * 2)
    _check_rows(r, codes, top[:, 0] / 127 / torch.sqrt(x.double().pow(2).mean(-1)))


def test_sum_in_place():
    """The C entry may write the sum over either summand."""
    g = _gen(3)
    x, res, w = (_rand(g, *s, dtype=torch.bfloat16) for s in ((7, 520), (7, 520), (520,)))
    want, total = rms_norm_int8(x, w, residual=res)
    for over in (0, 1):
        ops = [x.clone(), res.clone()]
        codes = torch.empty(7, 640, dtype=torch.int8, device=DEV)
        scales = torch.empty(7, device=DEV)
        _hip.check(_hip.lib().coda_rms_norm_int8(
            1, ops[0].data_ptr(), 520, ops[1].data_ptr(), 520, w.data_ptr(), 7, 520, 1e-6, ops[over].data_ptr(), 520,
            codes.data_ptr(), 640, scales.data_ptr(), _hip.stream_of(x)))
        assert torch.equal(ops[over], total) and torch.equal(codes, want.codes) and torch.equal(scales, want.scales)


@pytest.mark.parametrize("D", [9, 600])
def test_more_rows_than_a_launch(D):
    """Rows past 2^21, which a second launch takes, are the rows that they
    repeat."""
    g, M = _gen(D), (1 << 21) + 1405
    base, w = _rand(g, 1000, D, dtype=torch.bfloat16), _rand(g, D, dtype=torch.bfloat16)
    at = torch.arange(M, device=DEV) % 1000
    x = base[at]
    r, want = quantize_rows(x), quantize_rows(base)
    assert torch.equal(r.codes, want.codes[at]) and torch.equal(r.scales, want.scales[at])
    assert torch.equal(r.dequantize(), want.dequantize()[at])
    (r, total), (want, t0) = (rms_norm_int8(t, w, residual=t) for t in (x, base))
    assert torch.equal(r.codes, want.codes[at]) and torch.equal(r.scales, want.scales[at]) and torch.equal(total, t0[at])


# ---------------------------------------------------------------- product
def _int8(g, rows, K):
    """Plain codes of the whole range, and scales."""
    return (torch.randint(-127, 128, (rows, K), generator=g, device=DEV, dtype=torch.int8),
            torch.rand(rows, generator=g, device=DEV) * 0.01 + 1e-4)


def _check_product(y, a, sa, b, sb, bias):
    v = (a.double() @ b.double().t()) * sa.double()[:, None] * sb.double()[None]
    want = v if bias is None else v + bias.double()
    lim = want.abs() * (U + torch.finfo(y.dtype).eps / 2) * 1.001 + v.abs() * 3.01 * U + 2.0 ** -25
    assert ((y.double() - want).abs() <= lim).all()


SHAPES = [(1, 1, 1), (1, 4096, 6177), (2, 512, 16), (3, 100, 7), (16, 1024, 515), (17, 129, 64), (33, 2048, 1000),
          (64, 4096, 130), (65, 640, 257), (128, 1000, 2049), (129, 4096, 300), (200, 8192, 70), (255, 256, 255),
          (256, 128, 256), (257, 384, 513), (512, 1111, 777), (1000, 512, 1030), (1999, 300, 1029), (2049, 128, 2050)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,K,N", SHAPES)
def test_linear_int8(M, K, N, dtype):
    g = _gen(M + K + N)
    (a, sa), (b, sb) = _int8(g, M, K), _int8(g, N, K)
    x, w = Int8Rows.from_codes(a, sa, dtype), Int8Rows.from_codes(b, sb, dtype)
    bias = _rand(g, N, dtype=dtype) if (M + N) % 2 else None
    # (fp16 holds what these make only scaled down)
    if dtype == torch.float16:
        x, sa = Int8Rows(x.codes, x.scales / 256, K, dtype), sa / 256
    _check_product(linear_int8(x, w, bias), a, sa, b, sb, bias)


@pytest.mark.parametrize("K", [1, 128, 129, 300, 384, 512, 520, 640, 896, 1000, 1152])
@pytest.mark.parametrize("M,N", [(70, 500), (200, 1030), (128, 10305), (130, 9000), (250, 4100), (190, 8100)])
def test_shares_of_k(M, K, N):
    """Few and odd numbers of steps where several waves share K: some have one
    step more than others, or none."""
    g = _gen(K + M)
    (a, sa), (b, sb) = _int8(g, M, K), _int8(g, N, K)
    bias = _rand(g, N, dtype=torch.bfloat16)
    y = linear_int8(Int8Rows.from_codes(a, sa, torch.bfloat16), Int8Rows.from_codes(b, sb, torch.bfloat16), bias)
    _check_product(y, a, sa, b, sb, bias)


@pytest.mark.parametrize("M", [1, 40, 300])
def test_longest_sum(M):
    """Codes of 127 all along the longest row: just below 2^31."""
    K = 130944
    a, b = (torch.full((n, K), 127, dtype=torch.int8, device=DEV) for n in (M, 48))
    b[1::2] *= -1
    one = lambda n: torch.ones(n, device=DEV)  # noqa: E731
    y = linear_int8(Int8Rows(a, one(M), K, torch.float32), Int8Rows(b, one(48), K, torch.float32))
    want = torch.tensor(127 * 127 * K, dtype=torch.float64).float().item()
    assert (y[:, ::2] == want).all() and (y[:, 1::2] == -want).all()


@pytest.mark.parametrize("M", [2, 100, 118, 700])
def test_codes_of_any_layout(M):
    """Rows with gaps, rows off 16 bytes, one row for all tokens, leading
    dimensions: as dense codes."""
    g, K, N = _gen(M), 512, 200
    (a, sa), (b, sb) = _int8(g, M, K), _int8(g, N, K)
    w = Int8Rows(b, sb, K, torch.bfloat16)
    dense = linear_int8(Int8Rows(a, sa, K, torch.bfloat16), w)
    gap = torch.empty(M, K + 48, dtype=torch.int8, device=DEV)[:, 16:16 + K].copy_(a)
    off = torch.empty(M * K + 5, dtype=torch.int8, device=DEV)[5:].view(M, K).copy_(a)
    odd = torch.empty(M, K + 7, dtype=torch.int8, device=DEV)[:, :K].copy_(a)
    for c in (gap, off, odd):
        assert torch.equal(linear_int8(Int8Rows(c, sa, K, torch.bfloat16), w), dense)
    wide = torch.empty(N, 2 * K, dtype=torch.int8, device=DEV)[:, K:].copy_(b)
    far = torch.empty(M, 1 << 15, K, dtype=torch.int8, device=DEV)[:, 7].copy_(a) if M < 120 else a  # 16 MiB apart
    further = torch.empty(M, (1 << 15) + 1, K, dtype=torch.int8, device=DEV)[:, 7].copy_(a) if M < 120 else a
    for c in (far, further):
        assert torch.equal(linear_int8(Int8Rows(c, sa, K, torch.bfloat16), w), dense)
    scales = torch.stack([sb, sb], 1)[:, 0]
    assert torch.equal(linear_int8(Int8Rows(a, sa, K, torch.bfloat16), Int8Rows(wide, scales, K, torch.bfloat16)), dense)
    same = linear_int8(Int8Rows(a[:1].expand(M, K), sa[:1].expand(M), K, torch.bfloat16), w)
    assert torch.equal(same, dense[:1].expand(M, N))
    lead = linear_int8(Int8Rows(a.view(2, M // 2, K), sa.view(2, M // 2), K, torch.bfloat16), w)
    assert torch.equal(lead, dense.view(2, M // 2, N))
    assert linear_int8(Int8Rows(a[:0], sa[:0], K, torch.bfloat16), w).shape == (0, N)


@pytest.mark.parametrize("M", [1, 16, 60, 130, 400, 3000])
def test_a_row_is_its_own(M):
    """A token's result does not depend on the tokens beside it, whichever
    kernel the number of tokens takes, and is the same at every call."""
    g, K, N = _gen(9), 1024, 640
    (a, sa), (b, sb) = _int8(g, 3000, K), _int8(g, N, K)
    w = Int8Rows(b, sb, K, torch.bfloat16)
    run = lambda n: linear_int8(Int8Rows(a[:n], sa[:n], K, torch.bfloat16), w)  # noqa: E731
    y, whole = run(M), run(3000)
    assert torch.equal(y, whole[:M]) and torch.equal(run(M), y)


@pytest.mark.parametrize("M,K,N", [(33000, 130944, 64), (600000, 100, 4096)])
def test_offsets_past_32_bits(M, K, N):
    """4.3 GB of codes; 2.5 G values: the rows that they repeat."""
    g = _gen(M)
    rows = Int8Rows.from_codes(*_int8(g, 1000, K), torch.bfloat16)
    w = Int8Rows.from_codes(*_int8(g, N, K), torch.bfloat16)
    many = Int8Rows(rows.codes.repeat(M // 1000, 1), rows.scales.repeat(M // 1000), K, torch.bfloat16)
    y, want = linear_int8(many, w), linear_int8(rows, w)
    assert all(torch.equal(part, want) for part in y.view(-1, 1000, N))


@pytest.mark.parametrize("M", [3, 90, 1100])
def test_writes_nothing_else(M):
    """Behind and between the rows of the output: as it was."""
    g, K, N = _gen(M), 256, 77
    (a, sa), (b, sb) = _int8(g, M, K), _int8(g, N, K)
    for code, dt in enumerate((torch.float32, torch.bfloat16, torch.float16)):
        out = torch.full((M + 2, N + 5), 7.0, dtype=dt, device=DEV)
        _hip.check(_hip.lib().coda_linear_int8(code, a.data_ptr(), K, sa.data_ptr(), M, 0, b.data_ptr(), K, sb.data_ptr(), N,
                                               K, None, out[1, 2:].data_ptr(), N + 5, _hip.stream_of(a)))
        want = linear_int8(Int8Rows(a, sa, K, dt), Int8Rows(b, sb, K, dt))
        assert torch.equal(out[1:-1, 2:2 + N], want)
        out[1:-1, 2:2 + N] = 7.0
        assert (out == 7.0).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,K,N", [(1, 1, 1), (1, 4096, 6177), (2, 100, 7), (3, 127, 50), (5, 1000, 515), (16, 8192, 130),
                                   (16, 333, 2049), (17, 512, 64), (150, 200, 300), (1, 130, 8200), (4, 30001, 33)])
def test_tokens_as_they_come(M, K, N, dtype):
    """A float x: the bits of quantize_rows and the product of its rows, rows
    without a number among them."""
    g = _gen(M * K + N)
    x, q = _rand(g, M, K, dtype=dtype), quantize_rows(_rand(g, N, K, dtype=dtype))
    if M > 2:
        x[1], x[2, K // 2] = 0, float("inf")
    bias = _rand(g, N, dtype=dtype)
    for b in (None, bias):
        assert torch.equal(linear_int8(x, q, b).nan_to_num(7.0), linear_int8(quantize_rows(x), q, b).nan_to_num(7.0))
    if M > 2:
        y = linear_int8(x, q)
        assert not y[1].any() and y[2].isnan().all()
    wide = torch.full((M, K + 3), float("nan"), device=DEV, dtype=dtype)[:, 2:K + 2].copy_(x)
    for v in (wide, x.t().contiguous().t(), x.view(1, M, 1, K)):
        assert torch.equal(linear_int8(v, q).reshape(M, N).nan_to_num(7.0), linear_int8(x, q).nan_to_num(7.0))
    assert torch.equal(linear_int8(x[:1].expand(M, K), q), linear_int8(x[:1], q).expand(M, N))


# ---------------------------------------------------------------- together
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,L,D,N", [(1, 1, 512, 640), (3, 1, 1000, 515), (2, 150, 768, 1030), (5, 333, 256, 300)])
def test_a_block(B, L, D, N, dtype):
    """Norm with residual, product, quantised rows, product: as a block runs
    them, against the formulas in 64 bits on the values handed on."""
    g = _gen(B * L)
    x, res = _rand(g, B, L, D, dtype=dtype), _rand(g, B, L, D, dtype=dtype, std=2.0)
    w, w1, w2 = (1 + 0.2 * _rand(g, D)).to(dtype), _rand(g, N, D, dtype=dtype, std=D ** -0.5), _rand(g, D, N, std=N ** -0.5).to(dtype)
    q1, q2 = quantize_rows(w1), quantize_rows(w2)
    rows, s = rms_norm_int8(x, w, residual=res)
    h = linear_int8(rows, q1)
    again = quantize_rows(h)
    y = linear_int8(again, q2)
    assert y.shape == x.shape and h.shape == (B, L, N)
    f = lambda r: r.codes[..., :r.cols].reshape(-1, r.cols)  # noqa: E731
    _check_product(h.view(-1, N), f(rows), rows.scales.view(-1), f(q1), q1.scales, None)
    _check_product(y.view(-1, D), f(again), again.scales.view(-1), f(q2), q2.scales, None)
    # and near the products of the unrounded values: a code is off by half a
    # step, 1 / 254 of its row's largest value, and errors of one sign in all
    # of a row's products would add up to D times that
    full = s.double() * w.double() / torch.sqrt(s.double().pow(2).mean(-1, keepdim=True) + 1e-6)
    top, top1 = full.abs().amax(-1, keepdim=True), w1.double().abs().amax(-1)
    want = full @ w1.double().t()
    lim = (full.abs().sum(-1, keepdim=True) * top1 + w1.double().abs().sum(-1) * top) / 254 + D * top * top1 / 254 ** 2
    assert ((h.double() - want).abs() <= lim * 1.001 + want.abs() * torch.finfo(dtype).eps).all()


@pytest.mark.parametrize("M", [1, 64, 500])
def test_captured(M):
    """In a graph, replayed on other inputs with eager work in between."""
    g, D, N = _gen(M), 1024, 700
    x, res, w = _rand(g, M, D, dtype=torch.bfloat16), _rand(g, M, D, dtype=torch.bfloat16), _rand(g, D, dtype=torch.bfloat16)
    q = quantize_rows(_rand(g, N, D, dtype=torch.bfloat16))

    def run():
        rows, s = rms_norm_int8(x, w, residual=res)
        return s, linear_int8(rows, q), rows.dequantize()

    run()
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        out = run()
    torch.cuda.current_stream().wait_stream(side)
    for rep in range(3):
        x.copy_(_rand(g, M, D, dtype=torch.bfloat16))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, run()):
            assert torch.equal(a, b), f"replay {rep}"


def test_streams():
    """Two at once on streams of their own: each as it is alone."""
    g, D, N = _gen(4), 2048, 1500
    q = quantize_rows(_rand(g, N, D, dtype=torch.bfloat16))
    xs = [_rand(g, n, D, dtype=torch.bfloat16) for n in (40, 900)]
    want = [linear_int8(quantize_rows(x), q) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    got = [[], []]
    for _ in range(4):
        for i, (s, x) in enumerate(zip(streams, xs)):
            with torch.cuda.stream(s):
                got[i].append(linear_int8(quantize_rows(x), q))
    torch.cuda.synchronize()
    for ys, y in zip(got, want):
        assert all(torch.equal(a, y) for a in ys)


def test_refusals_on_the_device():
    x, w = torch.randn(4, 64, device=DEV), torch.ones(64, device=DEV)
    with pytest.raises(RuntimeError, match="weight"):
        rms_norm_int8(x, w[:63])
    with pytest.raises(RuntimeError, match="weight is"):
        rms_norm_int8(x, w.bfloat16())
    with pytest.raises(RuntimeError, match="residual"):
        rms_norm_int8(x, w, residual=x[:3])
    with pytest.raises(RuntimeError, match="negative"):
        rms_norm_int8(x, w, eps=-1.0)
    with pytest.raises(RuntimeError, match="rows of 1 to"):
        quantize_rows(torch.zeros(1, 32769, device=DEV))
    with pytest.raises(TypeError, match="dtype"):
        quantize_rows(x.double())
    q = quantize_rows(x)
    with pytest.raises(TypeError, match="Int8Rows"):
        linear_int8(q, x)
    with pytest.raises(RuntimeError, match="does not fit"):
        linear_int8(q, quantize_rows(x[:, :63]))
    with pytest.raises(RuntimeError, match="bias"):
        linear_int8(q, q, torch.zeros(4, device=DEV, dtype=torch.bfloat16))
    with pytest.raises(RuntimeError, match="int32"):
        long = torch.zeros(1, 131072, dtype=torch.int8, device=DEV)
        r = Int8Rows(long, w[:1], 131072, torch.float32)
        linear_int8(r, r)
