"""The 8-bit operators of coda_gqa_l, as cases to time and compare.

Kinds of case, each what a user's program calls in a row:

  norm    rms_norm_int8 with a residual, and the values that its codes stand
          for (Int8Rows.dequantize), as a block has them that hands the
          normalised tokens to a projection kept in full precision
  linear  linear_int8 on codes that are there already: the second and
          further projections of the same tokens
  rows    quantize_rows, then linear_int8: an output projection
  block   rms_norm_int8 with a residual, then linear_int8: a block's way
          into its attention

With own False the operators are computed from their formulas by elementary
torch operations: sums and products in fp32, the codes of fp32 rows in 64
bits (a quotient next to a half has to fall on the right side).

Values: activations with a few channels far above the others, as residual
streams have them; weights as nn.Linear draws them; norm weights about 1.
"""

import math
import os
import sys

import torch

own = False

DEV = "cuda:0"
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
PAD = 128  # codes of a row are followed by zeros up to a multiple of this


def _case(kind, M, K, N=0, dtype="bf16", bias=False):
    return dict(kind=kind, M=M, K=K, N=N, dtype=dtype, bias=bias)


def listed():
    return [
        # one user's next token on the 7B-shaped layer: latency
        dict(name="norm_1x4096", **_case("norm", 1, 4096)),
        # an odd batch of a small fp32 model whose width is no multiple of 64
        dict(name="norm_777x1000_f32", **_case("norm", 777, 1000, dtype="f32")),
        # two prompts of 8192 tokens on the 70B-shaped layer
        dict(name="norm_16384x8192", **_case("norm", 16384, 8192)),
        # q | k | v | lambda | gate of the 7B-shaped layer: one token, four streams of 8192
        dict(name="linear_1x4096_6177", **_case("linear", 1, 4096, 6177, bias=True)),
        dict(name="linear_32768x4096_6177", **_case("linear", 32768, 4096, 6177, bias=True)),
        # the 70B-shaped layer's output projection of two prompts
        dict(name="linear_16384x8192_8192", **_case("linear", 16384, 8192, 8192)),
        # a small fp32 model with biases, no size a multiple of anything
        dict(name="linear_333x1000_515_f32", **_case("linear", 333, 1000, 515, "f32", True)),
        # the output projection of a serving batch (70B shape) and of one prompt of no round length (7B shape)
        dict(name="rows_128x8192_8192", **_case("rows", 128, 8192, 8192)),
        dict(name="rows_1999x4096_4096", **_case("rows", 1999, 4096, 4096)),
        # the way into the attention: a serving batch of the 7B and one of the 70B shape, a half-precision prompt
        dict(name="block_64x4096_6177", **_case("block", 64, 4096, 6177, bias=True)),
        dict(name="block_128x8192_10305", **_case("block", 128, 8192, 10305, bias=True)),
        dict(name="block_500x2048_3105_f16", **_case("block", 500, 2048, 3105, "f16", True)),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("norm", "norm", "linear", "linear", "rows", "block", "block"))
    dtype = rng.choice(("bf16", "bf16", "bf16", "f16", "f32"))
    # tokens of a decode batch, or of prompts
    M = _log(rng, 1, 128) if rng.random() < 0.5 else _log(rng, 129, 16384)
    K = rng.choice((512, 1024, 2048, 4096, 4096, 8192, _log(rng, 64, 8192), _log(rng, 64, 8192)))
    if kind == "norm":
        return _case(kind, M, K, dtype=dtype)
    return _case(kind, M, K, rng.choice((512, 1024, 4096, 8192, _log(rng, 16, 10305), _log(rng, 512, 10305))) if
                 M * K <= 8192 * 8192 else _log(rng, 16, 8192), dtype, rng.random() < 0.5)


# ----------------------------------------------------------------- prepare
def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device=DEV)


def _tokens(gen, M, K, dtype, std, far):
    """(M, K) activations; a channel in 64 is `far` times the others."""
    x = _randn(gen, M, K).mul_(std)
    return x.mul_(1.0 + (far - 1.0) * (torch.rand(K, generator=gen, device=DEV) < 1 / 64)).to(dtype)


def _coded(x):
    """Codes (rows, K up to a multiple of PAD, zeros behind K) and scales."""
    K = x.shape[1]
    top = x.abs().amax(1)
    codes = torch.zeros(x.shape[0], -(-K // PAD) * PAD, dtype=torch.int8, device=DEV)
    codes[:, :K] = torch.round(x * (127.0 / top)[:, None]).to(torch.int8)
    return codes, top / 127.0


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    M, K, N, dt = case["M"], case["K"], case["N"], DTYPES[case["dtype"]]
    s = dict(case)
    if case["kind"] in ("norm", "block"):
        # a sublayer's output, the residual stream and the norm's weight
        s["x"], s["residual"] = _tokens(gen, M, K, dt, 0.4, 1.0), _tokens(gen, M, K, dt, 1.0, 12.0)
        s["weight"] = (1.0 + 0.2 * _randn(gen, K)).to(dt)
    elif case["kind"] == "rows":
        s["x"] = _tokens(gen, M, K, dt, 0.7, 3.0)
    else:
        s["a"], s["a_scales"] = _coded(_tokens(gen, M, K, torch.float32, 1.0, 6.0))
    if N:
        s["b"], s["b_scales"] = _coded((torch.rand(N, K, generator=gen, device=DEV) * 2.0 - 1.0) * K ** -0.5)
    s["bias"] = _randn(gen, N).mul_(0.5).to(dt) if case["bias"] else None
    return s


# ----------------------------------------------------------------- run
EPS = 1e-6


def _plain_codes(p, dt):
    """Codes of rows p and their largest magnitudes."""
    top = p.abs().amax(1, keepdim=True)
    if dt == torch.float32:
        p, top = p.double(), top.double()
    return torch.round(p * 127.0 / top), top


def _plain_norm(s):
    """(sum with the residual, codes, scales) of rms_norm_int8."""
    dt = s["x"].dtype
    total = (s["x"].float() + s["residual"].float()).to(dt)
    f = total.float()
    p, w = f, s["weight"].float()
    if dt == torch.float32:
        p, w = p.double(), w.double()
    codes, top = _plain_codes(p * w, dt)
    scales = top.float() * torch.rsqrt((f * f).mean(1, keepdim=True) + EPS) / 127.0
    return total, codes.float(), scales


def _plain_linear(s, codes, scales):
    y = (codes @ s["b"][:, :s["K"]].float().t()) * scales * s["b_scales"]
    if s["bias"] is not None:
        y = y + s["bias"].float()
    return y.to(DTYPES[s["dtype"]])


def _run_plain(s):
    kind, dt = s["kind"], DTYPES[s["dtype"]]
    if kind == "linear":
        return _plain_linear(s, s["a"][:, :s["K"]].float(), s["a_scales"][:, None])
    if kind == "rows":
        codes, top = _plain_codes(s["x"].float(), dt)
        return _plain_linear(s, codes.float(), top.float() / 127.0)
    total, codes, scales = _plain_norm(s)
    if kind == "norm":
        return total, (codes * scales).to(dt)
    return total, _plain_linear(s, codes, scales)


def _run_own(s):
    c = _package()
    kind, dt = s["kind"], DTYPES[s["dtype"]]
    w = c.Int8Rows(s["b"], s["b_scales"], s["K"], dt) if s["N"] else None
    if kind == "linear":
        return c.linear_int8(c.Int8Rows(s["a"], s["a_scales"], s["K"], dt), w, s["bias"])
    if kind == "rows":
        return c.linear_int8(c.quantize_rows(s["x"]), w, s["bias"])
    rows, total = c.rms_norm_int8(s["x"], s["weight"], EPS, residual=s["residual"])
    return total, rows.dequantize() if kind == "norm" else c.linear_int8(rows, w, s["bias"])


_pkg = None


def _package():
    global _pkg
    if _pkg is None:
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "coda-gqa-l_amd"))
        import coda_gqa_l
        _pkg = coda_gqa_l
    return _pkg


def run(state):
    if own:
        return _run_own(state)
    return _run_plain(state)


# ----------------------------------------------------------------- work, exact
def work(case):
    M, K, N, e = case["M"], case["K"], case["N"], DTYPES[case["dtype"]].itemsize
    kind = case["kind"]
    # x, residual and weight in, the sum out; or x in; or codes and scales in
    nbytes = {"norm": 3 * M * K * e + K * e, "block": 3 * M * K * e + K * e, "rows": M * K * e,
              "linear": M * K + 4 * M}[kind]
    flops = {"norm": 10, "block": 10, "rows": 4, "linear": 0}[kind] * M * K
    if kind == "norm":
        return {"bytes": nbytes + M * K * e, "flops": flops}
    return {"bytes": nbytes + N * K + 4 * N + M * N * e + (N * e if case["bias"] else 0),
            "flops": flops + 2 * M * N * K}


def exact(case, seed):
    s = prepare(case, seed)
    kind, dt, K = s["kind"], DTYPES[s["dtype"]], s["K"]
    if kind == "linear":
        a, sa = s["a"][:, :K].double(), s["a_scales"].double().unsqueeze(1)
    else:
        rows = s["x"].double()
        inv = torch.ones(rows.shape[0], 1, dtype=torch.float64, device=DEV)
        if kind != "rows":
            total = rows + s["residual"].double()
            h = total.to(dt).double()  # the norm is of the sum as it is kept
            inv = 1.0 / torch.sqrt(h.pow(2).sum(1, keepdim=True) / K + EPS)
            rows = h * s["weight"].double()
        largest = rows.abs().max(dim=1, keepdim=True).values
        a = torch.round(rows / largest * 127.0)
        sa = largest * inv / 127.0
    if kind == "norm":
        return total, a * sa
    y = torch.matmul(a, s["b"][:, :K].double().t()) * (sa * s["b_scales"].double().unsqueeze(0))
    if s["bias"] is not None:
        y = y + s["bias"].double().unsqueeze(0)
    return y if kind in ("linear", "rows") else (total, y)
