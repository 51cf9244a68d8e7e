"""The layers on 8-bit projections: the front end against its formulas in 64
bits, and prompts, steps and adapters against the parts that they are made of
(front end, attention on its outputs, quantised heads times quantised o_proj)."""
import copy
import io

import pytest
import torch
import torch.nn as nn

import coda_gqa_l
from coda_gqa_l import Int8Rows, linear_int8, quantize_rows, rms_norm_int8, state_io

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
FIELDS = ("k_buf", "v_buf", "allowed", "g_recent", "mem_last_exact", "_exact_v_norm", "_sum_lf_k_norm")


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _rand(g, *shape, dtype=torch.float32, std=1.0):
    return (torch.randn(*shape, generator=g, device=DEV) * std).to(dtype)


def _settle(m, seed):
    g = _gen(seed)
    with torch.no_grad():
        for lin in (m.q_proj, m.k_proj, m.v_proj, m.o_proj, m.lambda_proj):
            lin.weight.uniform_(-lin.in_features ** -0.5, lin.in_features ** -0.5, generator=g)
        m.lambda_proj.bias.copy_(_rand(g, m.num_heads, std=0.5) - 1.0)
        m.theta.copy_(m.theta + _rand(g, *m.theta.shape, std=0.1))
        if hasattr(m, "write_proj"):
            m.write_proj.weight.copy_(_rand(g, 1, m.embed_dim, std=0.7 * m.embed_dim ** -0.5))
    return m


def _bounded(dtype=torch.bfloat16, D=512, H=8, Hkv=2, seed=1, **kw):
    kw = dict(dict(window=32, num_landmarks_exact=16, num_landmarks_summary=16), **kw)
    m = coda_gqa_l.CoDAGQALandmarkPerf2(embed_dim=D, num_heads=H, num_kv_heads=Hkv, **kw)
    return _settle(m.to(DEV, dtype).eval(), seed).use_int8_projections()


def _unbounded(dtype=torch.bfloat16, D=512, H=8, Hkv=2, seed=1, **kw):
    m = coda_gqa_l.CoDAGQA(embed_dim=D, num_heads=H, num_kv_heads=Hkv, **kw)
    return _settle(m.to(DEV, dtype).eval(), seed).use_int8_projections()


def _state(m, B, dtype, seed=3):
    torch.manual_seed(seed)
    return m.init_state(batch_size=B, device=DEV, dtype=dtype)


def _same_state(a, b):
    for f in FIELDS:
        x, y = getattr(a, f), getattr(b, f)
        assert (x is None) == (y is None) and (x is None or torch.equal(x, y)), f
    assert (a.pos, a.recent_idx, a.recent_filled) == (b.pos, b.recent_idx, b.recent_filled)


def _out(m, heads):
    """o_proj in 8 bits from the public operators."""
    B, L = heads.shape[:2]
    return linear_int8(quantize_rows(heads.reshape(B, L, -1)), quantize_rows(m.o_proj.weight), m.o_proj.bias)


# ---------------------------------------------------------------- front end
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,L,D,H,Hkv,inter,gate", [
    (1, 1, 512, 8, 2, True, True), (5, 1, 512, 8, 2, False, True), (33, 1, 320, 10, 5, True, False),
    (128, 1, 256, 4, 1, False, True), (2, 100, 512, 4, 4, True, True), (3, 77, 320, 5, 1, False, True),
    (1, 999, 768, 12, 4, False, False), (2, 300, 240, 20, 4, True, False), (3, 150, 240, 20, 5, False, False),
    (2, 2, 240, 20, 4, False, False), (2, 4097, 256, 4, 2, True, True), (4, 4100, 768, 6, 3, False, True),
])
@torch.no_grad()
def test_front(B, L, D, H, Hkv, inter, gate, dtype):
    Dh = D // H
    if gate:
        m = _bounded(dtype, D, H, Hkv, rope_interleaved=inter)
    else:
        m = _unbounded(dtype, D, H, Hkv, rope_interleaved=inter)
    g0 = _gen(B + L)
    for lin in (m.q_proj, m.k_proj):  # biases, as some models have them
        lin.bias = nn.Parameter(_rand(g0, lin.out_features, dtype=dtype, std=0.3))
    x = _rand(g0, B, L, D, dtype=dtype)
    r = quantize_rows(x)
    q, k, v, g, lam, cos, sin = m._front_int8(r, 11)
    again = m._front_int8(x, 11)
    for a, b in zip((q, k, v, lam), (again[0], again[1], again[2], again[4])):
        assert torch.equal(a, b)
    eps = torch.finfo(dtype).eps
    a64 = r.codes[..., :D].double()

    def linear(lin):
        w = quantize_rows(lin.weight)
        y = (a64 @ w.codes[:, :D].double().t()) * r.scales.double()[..., None] * w.scales.double()
        err = 3.01 * U * y.abs()
        if lin.bias is not None:
            y = y + lin.bias.double()
        # the linear's own rounding, and the fp32 ones before it
        return y, err + y.abs() * (U + eps / 2) * 1.001

    for got, lin, heads in ((q, m.q_proj, H), (v, m.v_proj, Hkv)):
        y, err = linear(lin)
        assert ((got.permute(0, 2, 1, 3).reshape(B, L, heads * Dh).double() - y).abs() <= err).all()
    # k: two products and their sum, a rounding each, of values off by err
    y, err = (t.view(B, L, Hkv, Dh) for t in linear(m.k_proj))
    c, s = (t.double()[None, :, None, :] for t in (cos, sin))
    pick = (lambda t: (t[..., 0::2], t[..., 1::2])) if inter else (lambda t: (t[..., :Dh // 2], t[..., Dh // 2:]))
    (y0, y1), (e0, e1) = pick(y), pick(err)
    got0, got1 = pick(k.permute(0, 2, 1, 3).double())
    for got, a, b, ea, eb, sign in ((got0, y0, y1, e0, e1, -1), (got1, y1, y0, e1, e0, 1)):
        want, size = a * c + sign * b * s, (a * c).abs() + (b * s).abs()
        lim = ea * c.abs() + eb * s.abs() + (size * eps / 2 + (want.abs() + size * eps / 2) * eps / 2) * 1.01
        assert ((got - want).abs() <= lim).all()
    # sigmoids: slope at most 1/4; fp32 expf and division within 8 ulp
    for got, lin in ((lam.permute(0, 2, 1), m.lambda_proj),) + (((g[..., None], m.write_proj),) if gate else ()):
        y, err = linear(lin)
        want = torch.sigmoid(y)
        assert ((got.double() - want).abs() <= err / 4 + want * (eps / 2 + 8 * U) * 1.01).all()
    assert gate or g is None


# ---------------------------------------------------------------- bounded layer
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,L,fresh,policy", [(1, 70, True, "gated"), (2, 200, True, "gated"), (3, 130, False, "gated"),
                                              (2, 100, True, "none")])
@torch.no_grad()
def test_prompts_are_their_parts(B, L, fresh, policy, dtype):
    m = _bounded(dtype, write_policy=policy)
    g = _gen(L)
    a, b, c = (_state(m, B, dtype) for _ in range(3))
    if not fresh:
        x0 = _rand(g, B, 90, 512, dtype=dtype)
        for st in (a, b, c):
            m.prefill_chunked(x0, st, block_size=32)
    x = _rand(g, B, L, 512, dtype=dtype)
    y, a = m.prefill_chunked(x, a, block_size=32)
    q, k, v, gate, lam, cos, sin = m._front(x, int(b.pos))
    if policy == "none":
        assert (gate == 1).all()
    want = _out(m, m.prefill_core(q, k, v, gate, lam, cos, sin, b, block_size=32))
    assert torch.equal(y, want)
    _same_state(a, b)
    # tokens that arrive in 8 bits
    y2, c = m.prefill_chunked(quantize_rows(x), c, block_size=32)
    assert torch.equal(y2, y)
    _same_state(c, a)
    assert m.prefill_chunked(x[:, :0], a)[0].shape == (B, 0, 512)
    assert m.prefill_chunked(quantize_rows(x), c, block_size=32, return_outputs=False)[0] is None


@pytest.mark.parametrize("B,dtype,policy", [(1, torch.bfloat16, "gated"), (3, torch.float32, "gated"),
                                            (70, torch.bfloat16, "gated"), (130, torch.bfloat16, "none")])
@torch.no_grad()
def test_steps(B, dtype, policy):
    """The cached step, the general one, steps on 8-bit tokens and the parts:
    the same bits, from an empty ring over the steady state."""
    m = _bounded(dtype, write_policy=policy)
    g = _gen(B)
    sts = [_state(m, B, dtype) for _ in range(4)]
    x0 = _rand(g, B, 27, 512, dtype=dtype)
    for st in sts:
        m.prefill_chunked(x0, st, block_size=32)
    n = copy.deepcopy(m)  # never the cached step
    n._step_fast = lambda *args: None
    fast = 0
    for i in range(14):
        x = _rand(g, B, 1, 512, dtype=dtype)
        ys = [m.step(x, sts[0])[0], n.step(x, sts[1])[0], n.step(quantize_rows(x), sts[2])[0]]
        q, k, v, gate, lam, cos, sin = n._front(x, int(sts[3].pos))
        ys.append(_out(m, n.decode_step_core(q, k, v, gate.reshape(B), lam, sts[3], cos, sin)))
        for y in ys[1:]:
            assert torch.equal(y, ys[0]), i
        fast += m.__dict__.get("_fast") is not None
    for st in sts[1:]:
        _same_state(st, sts[0])
    assert fast > 4
    # the cached step on 8-bit tokens, and an odd view of them
    x = _rand(g, B, 1, 512, dtype=dtype)
    r = quantize_rows(x)
    odd = torch.empty(B * 512 + 3, dtype=torch.int8, device=DEV)[3:].view(B, 1, 512).copy_(r.codes)
    want = n.step(x, sts[1])[0]
    assert torch.equal(m.step(r, sts[0])[0], want)
    assert torch.equal(n.step(x, sts[1])[0], m.step(Int8Rows(odd, r.scales, 512, dtype), sts[0])[0])
    _same_state(sts[0], sts[1])


@torch.no_grad()
def test_partial_steps():
    m = _bounded()
    x = _rand(_gen(1), 2, 1, 512, dtype=torch.bfloat16)
    st, ref = _state(m, 2, torch.bfloat16), _state(m, 2, torch.bfloat16)
    for s in (st, ref):
        m.prefill_chunked(_rand(_gen(2), 2, 60, 512, dtype=torch.bfloat16), s, block_size=32)
    q, k, v, g, lam, cos, sin = m._front(x, int(ref.pos))
    want = _out(m, m.decode_attend_core(q, lam, ref, cos, sin))
    y, _ = m.step(x, st, write_cache=False)
    assert torch.equal(y, want)
    _same_state(st, ref)
    y, _ = m.step(quantize_rows(x), st, attend=False)
    m._write_one(ref, k_new=k, v_new=v, g_new=g)
    assert not y.any() and y.shape == (2, 1, 512) and y.dtype == torch.bfloat16
    _same_state(st, ref)


@torch.no_grad()
def test_parameters_that_change():
    """A counted change is seen; one through .data after
    drop_parameter_copies(); off again: the float layer's bits."""
    m = _bounded()
    plain = copy.deepcopy(m).use_int8_projections(False)
    st = _state(m, 2, torch.bfloat16)
    g = _gen(5)
    m.prefill_chunked(_rand(g, 2, 60, 512, dtype=torch.bfloat16), st, block_size=32)
    x = _rand(g, 2, 1, 512, dtype=torch.bfloat16)

    def run(layer):
        return layer.step(x, state_io.deep_copy_state(st))[0]

    ys = [run(m), run(m)]
    assert torch.equal(*ys)
    for name in ("q_proj", "v_proj", "o_proj"):
        for counted in (True, False):
            w = getattr(m, name).weight
            if counted:
                w.mul_(1.5)
            else:
                w.data *= 1.5
                m.drop_parameter_copies()
            y = run(m)
            assert not torch.equal(y, ys[-1])
            assert torch.equal(y, run(copy.deepcopy(m)))
            ys.append(y)
            getattr(plain, name).weight.copy_(w)
    assert torch.equal(run(m.use_int8_projections(False)), run(plain))
    # copies and saves carry the choice, not the codes
    m.use_int8_projections()
    y = run(m)
    buf = io.BytesIO()
    torch.save(m, buf)
    buf.seek(0)
    n = torch.load(buf, weights_only=False)  # written above
    assert n.int8_projections and "_int8_made" not in n.__dict__ and torch.equal(run(n), y)


@torch.no_grad()
def test_refused():
    m = _bounded()
    st = _state(m, 1, torch.bfloat16)
    x = _rand(_gen(1), 1, 4, 512, dtype=torch.bfloat16)
    m.use_int8_projections(False)
    with pytest.raises(RuntimeError, match="use_int8_projections"):
        m.prefill_chunked(quantize_rows(x), st)
    m.use_int8_projections()
    with pytest.raises(RuntimeError, match="not \\(B, L, 512\\)"):
        m._front_int8(quantize_rows(x[..., :500]), 0)
    # a steady state, then tokens of another width, or an o_proj bias of another type
    m.prefill_chunked(_rand(_gen(2), 1, 60, 512, dtype=torch.bfloat16), st, block_size=32)
    m.step(x[:, :1], st)
    for bad in (x[:, :1, :500], quantize_rows(x[:, :1, :500]), torch.cat([x[:, :1]] * 2, 2)):
        with pytest.raises(RuntimeError, match="not \\(B, L, 512\\)"):
            m.step(bad, st)
    m.o_proj.bias = nn.Parameter(torch.zeros(512, device=DEV))
    with pytest.raises(RuntimeError, match="bias"):
        m.step(x[:, :1], st)
    m.o_proj.bias = None
    m.step(x[:, :1], st)
    h = m.k_proj.register_forward_hook(lambda *a: None)
    with pytest.raises(RuntimeError, match="k_proj to be a plain"):
        m.prefill_chunked(x, st)
    h.remove()
    m.v_proj = nn.Sequential(m.v_proj)
    with pytest.raises(Exception, match="v_proj"):
        m.prefill_chunked(x, st)
    half = _bounded().half()
    with pytest.raises(RuntimeError, match="dtype"):
        half._front_int8(x.half(), 0)


@torch.no_grad()
@pytest.mark.parametrize("name", ["q_proj", "write_proj", "o_proj"])
def test_hooks_between_steps(name):
    """A hook, or a forward of its own, that a projection gets once steps run
    from descriptors is refused, and steps go on without it."""
    m = _bounded()
    st = _state(m, 1, torch.bfloat16)
    g = _gen(3)
    m.prefill_chunked(_rand(g, 1, 60, 512, dtype=torch.bfloat16), st, block_size=32)
    x = _rand(g, 1, 1, 512, dtype=torch.bfloat16)
    m.step(x, st)
    m.step(x, st)
    lin = getattr(m, name)
    for add, remove in ((lambda: lin.register_forward_hook(lambda *a: None), lambda h: h.remove()),
                        (lambda: lin.register_forward_pre_hook(lambda *a: None), lambda h: h.remove()),
                        (lambda: setattr(lin, "forward", lambda t: t), lambda h: delattr(lin, "forward"))):
        pos = int(st.pos)
        h = add()
        with pytest.raises(RuntimeError, match=name + " to be a plain"):
            m.step(x, st)
        assert int(st.pos) == pos
        remove(h)
        m.step(x, st)


# ---------------------------------------------------------------- unbounded layer
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,L,past,causal", [(1, 1, 0, True), (2, 65, 0, True), (1, 300, 0, False), (2, 3, 50, False),
                                             (3, 1, 120, False), (2, 20, 40, False), (200, 1, 30, False),
                                             (70, 2, 30, False)])
@torch.no_grad()
def test_unbounded(B, L, past, causal, dtype):
    m = _unbounded(dtype)
    g = _gen(L + past)
    x = _rand(g, B, L, 512, dtype=dtype)
    kv = tuple(_rand(g, B, 2, past, 64, dtype=dtype) for _ in range(2)) if past else None
    y, (k, v) = m(x, is_causal=causal, past_key_value=kv)
    q, kn, vn, _, lam, cos, sin = m._front_int8(quantize_rows(x), past)
    ks, vs = (torch.cat([p, n], 2) if past else n for p, n in zip(kv or (None, None), (kn, vn)))
    assert torch.equal(k, ks) and torch.equal(v, vs)
    heads = m.attention_core(q, ks, vs, lam, cos, sin, causal=2 if causal else 0)
    want = _out(m, heads)
    if dtype == torch.bfloat16 and past and L * 4 <= 8 and B * L <= 128:
        # another attention kernel: heads within the layer's bound, and codes
        # of heads that differ by it
        assert (y.float() - want.float()).abs().max() <= 4e-2 * want.float().abs().max()
    else:
        assert torch.equal(y, want)
    y8, (k8, _) = m(quantize_rows(x), is_causal=causal, past_key_value=kv)
    assert torch.equal(y8, y) and torch.equal(k8, k)


# ---------------------------------------------------------------- together
class _Attn(nn.Module):
    def __init__(self, D, H, Hkv):
        super().__init__()
        Dh = D // H
        self.q_proj, self.k_proj = nn.Linear(D, D, bias=True), nn.Linear(D, Hkv * Dh, bias=True)
        self.v_proj, self.o_proj = nn.Linear(D, Hkv * Dh, bias=False), nn.Linear(D, D, bias=False)
        self.num_heads, self.num_key_value_heads, self.head_dim = H, Hkv, Dh


@pytest.mark.parametrize("bounded", [True, False])
@torch.no_grad()
def test_adapter_behind_a_norm(bounded):
    """A block's way through an adapter: norm with residual in 8 bits, the
    layer on its rows, the sum with the residual; prompt, then tokens."""
    torch.manual_seed(0)
    ad = coda_gqa_l.LlamaCoDAAdapter.from_llama_attention(_Attn(512, 8, 2).to(DEV, torch.bfloat16), bounded=bounded,
                                                          head_norm_mode="full", rope_interleaved=True, block_size=32,
                                                          **(dict(window=32, num_landmarks_exact=16,
                                                                  num_landmarks_summary=16) if bounded else {}))
    ad = ad.eval().use_int8_projections()
    other = copy.deepcopy(ad)
    g = _gen(3)
    w = (1 + 0.1 * _rand(g, 512)).bfloat16()
    for st in range(2):
        torch.manual_seed(st)
        for L in (50, 1, 1) if bounded else (50, 7):
            x, res = _rand(g, 2, L, 512, dtype=torch.bfloat16), _rand(g, 2, L, 512, dtype=torch.bfloat16)
            rows, s = rms_norm_int8(x, w, residual=res)
            assert torch.equal(s, x + res)
            if bounded and ad.get_state() is None:
                init = ad.init_inference_state(2, torch.device(DEV), torch.bfloat16)
                other.set_state(state_io.deep_copy_state(init))
            y, _ = ad(rows)
            want, _ = other(Int8Rows(rows.codes.clone(), rows.scales.clone(), 512, torch.bfloat16))
            assert y.shape == (2, L, 512) and torch.isfinite(y.float()).all() and torch.equal(y, want)


@torch.no_grad()
def test_captured():
    """Front end and o_proj of a layer in a graph, as its first call."""
    for first in (True, False):
        m, plain = _bounded(), _bounded()
        g = _gen(9)
        x = _rand(g, 3, 1, 512, dtype=torch.bfloat16)
        if not first:
            m._front(x, 5)
            m._out_proj(x)
        side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
            out = (*m._front(x, 77)[:5], m._out_proj(x))
        torch.cuda.current_stream().wait_stream(side)
        for rep in range(3):
            x.copy_(_rand(g, 3, 1, 512, dtype=torch.bfloat16))
            graph.replay()
            torch.cuda.synchronize()
            for a, b in zip(out, (*plain._front(x, 77)[:5], plain._out_proj(x))):
                assert torch.equal(a, b), (first, rep)
            m.prefill_chunked(_rand(g, 1, 400, 512, dtype=torch.bfloat16), _state(m, 1, torch.bfloat16), block_size=32)
            junk = [torch.full((1 << n,), float("nan"), device=DEV) for n in range(8, 22)]
            del junk


@torch.no_grad()
def test_streams():
    """The codes made on one stream, used on another at once; steps of two
    states on streams of their own."""
    m, ref = _bounded(), _bounded()
    g = _gen(11)
    x = _rand(g, 2, 1, 512, dtype=torch.bfloat16)
    sts = [_state(m, 2, torch.bfloat16) for _ in range(2)]
    x0 = _rand(g, 2, 70, 512, dtype=torch.bfloat16)
    for st in sts:
        ref.prefill_chunked(x0, st, block_size=32)
    want_st = [state_io.deep_copy_state(st) for st in sts]
    want = [[ref.step(x, st)[0] for _ in range(3)] for st in want_st]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in sts], [[], []]
    for _ in range(3):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(m.step(x, sts[i])[0])
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert all(torch.equal(u, v) for u, v in zip(a, b))

