"""Rows in 8 bits: what is refused before any GPU call, and their layout."""
import pytest
import torch

import coda_gqa_l
from coda_gqa_l import Int8Rows, _hip, linear_int8


def test_layout_of_rows():
    c, s = torch.ones(2, 3, 100, dtype=torch.int8), torch.ones(2, 3)
    r = Int8Rows.from_codes(c, s, torch.bfloat16)
    assert r.codes.shape == (2, 3, 128) and r.shape == (2, 3, 100) and r.cols == 100 and not r.codes[..., 100:].any()
    assert Int8Rows.from_codes(torch.ones(4, 256, dtype=torch.int8), torch.ones(4), torch.float32).codes.shape == (4, 256)


@pytest.mark.parametrize("codes,scales,cols,dtype,error", [
    (torch.zeros(2, 100, dtype=torch.int8), torch.zeros(2), 100, torch.float32, "last size must be 128"),
    (torch.zeros(2, 256, dtype=torch.int8), torch.zeros(2), 100, torch.float32, "last size must be 128"),
    (torch.zeros(2, 128, dtype=torch.int8), torch.zeros(3), 128, torch.float32, "scales"),
    (torch.zeros(2, 128, dtype=torch.int8), torch.zeros(2, 1), 128, torch.float32, "scales"),
    (torch.zeros(2, 128, dtype=torch.uint8), torch.zeros(2), 128, torch.float32, "int8"),
    (torch.zeros(2, 128, dtype=torch.int8), torch.zeros(2).double(), 128, torch.float32, "int8"),
    (torch.zeros(2, 128, dtype=torch.int8), torch.zeros(2), 0, torch.float32, "last size"),
    (torch.zeros(2, 0, dtype=torch.int8), torch.zeros(2), 0, torch.float32, "last size"),
])
def test_rows_refused(codes, scales, cols, dtype, error):
    with pytest.raises(RuntimeError, match=error):
        Int8Rows(codes, scales, cols, dtype)


def test_other_types_refused():
    with pytest.raises(TypeError, match="dtype"):
        Int8Rows(torch.zeros(2, 128, dtype=torch.int8), torch.zeros(2), 128, torch.int32)


def test_no_host_path():
    x = torch.zeros(2, 128)
    r = Int8Rows(torch.zeros(2, 128, dtype=torch.int8), torch.zeros(2), 128, torch.float32)
    for call in (lambda: coda_gqa_l.quantize_rows(x), lambda: coda_gqa_l.rms_norm_int8(x, x[0]),
                 lambda: coda_gqa_l.linear_int8(r, r), lambda: coda_gqa_l.linear_int8(x, r), r.dequantize):
        with pytest.raises(RuntimeError, match="HIP devices only"):
            call()


P = 4096  # an address that no refused call reads


@pytest.mark.parametrize("args,error", [
    ((9, P, 64, 4, 64, P, 128, P), "dtype"),
    ((1, P, 64, -1, 64, P, 128, P), "sizes"),
    ((1, P, 64, 4, 0, P, 128, P), "sizes"),
    ((1, P, 64, 4, 64, P, 64, P), "hold D=64"),
    ((1, P, 64, 4, 64, P + 4, 128, P), "16-byte"),
    ((1, P, 64, 4, 64, P, 136, P), "16-byte"),
    ((1, P, 64, 4, 64, None, 128, P), "null"),
    ((1, None, 64, 4, 64, P, 128, P), "null"),
    ((1, P, 64, 4, 64, P, 128, None), "null"),
])
def test_quantize_rows_entry(args, error):
    L = _hip.lib()
    assert L.coda_quantize_rows(*args, None) == 1
    assert error in L.coda_last_error().decode()


def test_too_long_a_row_is_not_built():
    L = _hip.lib()
    assert L.coda_quantize_rows(1, P, 40000, 1, 40000, P, 40064, P, None) == _hip.CODA_EUNSUP


@pytest.mark.parametrize("change,error", [
    (dict(weight=None), "null"), (dict(sum_out=None), "null"), (dict(eps=-1.0), "negative"),
    (dict(eps=float("nan")), "negative"), (dict(dtype=5), "dtype"),
])
def test_rms_norm_entry(change, error):
    a = dict(dtype=1, x=P, x_sm=64, residual=P, r_sm=64, weight=P, rows=2, D=64, eps=1e-6, sum_out=P, s_sm=64, codes=P,
             c_sm=128, scales=P)
    a.update(change)
    L = _hip.lib()
    assert L.coda_rms_norm_int8(*a.values(), None) == 1
    assert error in L.coda_last_error().decode()


@pytest.mark.parametrize("change,error", [
    (dict(K=64), "multiple of 128"), (dict(K=131072), "int32"), (dict(K=0), "sizes"), (dict(n_feat=0), "sizes"),
    (dict(M=-1), "sizes"), (dict(x=P + 1), "16-byte"), (dict(w_sm=130), "16-byte"), (dict(w=None), "null"),
    (dict(x=None), "null"), (dict(out=None), "output"), (dict(o_sm=9), "output"), (dict(dtype=3), "dtype"),
    (dict(x_sm=-128), "16-byte"), (dict(x_sm=(1 << 24) + 16), "apart at most"), (dict(w_sm=1 << 25), "apart at most"),
    (dict(x_scales=None, M=5), "at most 4"), (dict(x_scales=None, D=129), "129 elements"),
    (dict(x_scales=None, D=0), "0 elements"), (dict(x_scales=None, x=None), "null"),
])
def test_linear_entry(change, error):
    a = dict(dtype=1, x=P, x_sm=128, x_scales=P, M=3, D=128, w=P, w_sm=128, w_scales=P, n_feat=10, K=128, bias=None, out=P,
             o_sm=10)
    a.update(change)
    L = _hip.lib()
    assert L.coda_linear_int8(*a.values(), None) == 1
    assert error in L.coda_last_error().decode()


@pytest.mark.parametrize("change", [dict(M=(1 << 30) + 1), dict(n_feat=(1 << 30) + 1, o_sm=1 << 31)])
def test_too_many_rows_of_a_product(change):
    a = dict(dtype=1, x=P, x_sm=128, x_scales=P, M=3, D=128, w=P, w_sm=128, w_scales=P, n_feat=10, K=128, bias=None, out=P,
             o_sm=10)
    a.update(change)
    L = _hip.lib()
    assert L.coda_linear_int8(*a.values(), None) == 2
    assert "2^30" in L.coda_last_error().decode()


def test_more_rows_than_32_bits_count():
    n = 1 << 31
    r = Int8Rows(torch.zeros(1, 128, dtype=torch.int8).expand(n, 128), torch.zeros(1).expand(n), 100, torch.float32)
    for call in (r.dequantize, lambda: linear_int8(r, r), lambda: linear_int8(torch.zeros(1, 100), r)):
        with pytest.raises(RuntimeError, match="2147483648 rows"):
            call()


@pytest.mark.parametrize("change,error", [
    (dict(dtype=2), "dtype"), (dict(Dh=6), "sizes"), (dict(M=-1), "sizes"), (dict(q=None), "missing"),
    (dict(bias=P + 4), "16-byte"), (dict(g=None), "missing"), (dict(k=P + 2), "8-byte"), (dict(x_sm=100), "16-byte"),
])
def test_project_entry(change, error):
    d = _hip.ProjDesc()
    for n, v in dict(dict(dtype=1, M=2, L=1, H=2, Hkv=1, Dh=64, gate=1, x=P, x_sm=128, w=P, bias=P, rope_cos=P, rope_sin=P,
                          q=P, q_sm=128, k=P, k_sm=64, v=P, v_sm=64, lam=P, lam_sm=2, g=P), **change).items():
        setattr(d, n, v)
    L = _hip.lib()
    assert L.coda_project_int8(d, P, P, 128, 128, None, None) == 1
    assert error in L.coda_last_error().decode()
    assert L.coda_project_int8(None, P, P, 128, 128, None, None) == 1


@pytest.mark.parametrize("dim,params,error", [
    (dict(M=129), dict(inv_freq=P, rope_cos=P, rope_sin=P), "at most 128"),
    (dict(), dict(inv_freq=P, rope_cos=P), "RoPE tables"),
    (dict(), dict(inv_freq=P, rope_cos=P, rope_sin=P, inv_dtype=2), "RoPE tables"),
    (dict(), dict(inv_freq=P, rope_cos=P, rope_sin=P, p0=1 << 24), "2^24"),
    (dict(), dict(theta=P, theta_cos=P), "theta tables"),
])
def test_project_entry_tables(dim, params, error):
    d, p = _hip.ProjDesc(), _hip.ProjParams()
    for n, v in dict(dict(dtype=1, M=2, L=1, H=2, Hkv=1, Dh=64, gate=1, x=P, x_sm=128, w=P, bias=P, rope_cos=P, rope_sin=P,
                          q=P, q_sm=128, k=P, k_sm=64, v=P, v_sm=64, lam=P, lam_sm=2, g=P), **dim).items():
        setattr(d, n, v)
    for n, v in params.items():
        setattr(p, n, v)
    L = _hip.lib()
    assert L.coda_project_int8(d, P, P, 128, 128, p, None) == 1
    assert error in L.coda_last_error().decode()


def _layer():
    m = coda_gqa_l.CoDAGQA(embed_dim=128, num_heads=4, num_kv_heads=2).bfloat16().eval()
    return m.use_int8_projections()


class _Mine(torch.nn.Linear):
    pass


class _Weight(torch.nn.Parameter):
    pass


@pytest.mark.parametrize("change", [
    lambda m: m.q_proj.register_forward_hook(lambda *a: None),
    lambda m: m.o_proj.register_forward_pre_hook(lambda *a: None),
    lambda m: setattr(m.k_proj, "forward", lambda x: x),
    lambda m: setattr(m, "v_proj", _Mine(128, 64)),
    lambda m: setattr(m.lambda_proj, "weight", _Weight(m.lambda_proj.weight.detach().clone())),
    lambda m: setattr(m, "q_proj", torch.nn.Linear(128, 64, bias=False)),
    lambda m: setattr(m, "o_proj", torch.nn.Linear(64, 128, bias=False)),
    lambda m: torch.nn.utils.parametrize.register_parametrization(m.q_proj, "weight", torch.nn.Identity()),
])
def test_only_plain_projections(change):
    import torch.nn.utils.parametrize  # noqa: F401
    m = _layer()
    assert len(m._int8_linears()) == 5
    change(m)
    with pytest.raises(RuntimeError, match="plain nn.Linear"):
        m._int8_linears()


def test_hooks_on_every_module():
    m = _layer()
    h = torch.nn.modules.module.register_module_forward_hook(lambda *a: None)
    try:
        with pytest.raises(RuntimeError, match="plain nn.Linear"):
            m._int8_linears()
    finally:
        h.remove()
    assert len(m._int8_linears()) == 5
