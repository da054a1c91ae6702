"""Rotary positions and the q / k norms with the rotation, against the formulas in 64 bits.

Bounds.  The result is rounded once to 16 bits: half a step, eps / 2 of the value (fp16: and 2^-25 where it is subnormal).  In
front of that the kernels work in fp32: the reduced angle, at most pi, is off by 2^-23 when it becomes fp32, __sinf and __cosf
by 2^-21.19 at most from minus pi to pi, and a turned value adds two products (2^-24 each): below 2^-20 of |a| + |b| for the
pair (a, b).  A norm's 1 / rms is off by half of its sum's error (8 + log2(D / 8) roundings of terms of one sign) and two ulp:
below 2^-20 of its value, so that a normed pair gets 2^-19."""
import itertools
import math

import pytest
import torch

import forgetting_transformer_b200 as fox

pytestmark = pytest.mark.gpu


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    return 2.0 ** -25 if dtype == torch.float16 else 0.0


def pairs(half, interleaved, device):
    i = torch.arange(half, device=device)
    return (2 * i, 2 * i + 1) if interleaved else (i, i + half)


def turn64(x, angles, interleaved, scale=1.0, sign=1.0):
    """x (..., D) in 64 bits; angles (..., half), broadcast over x's leading axes."""
    a, b = pairs(angles.shape[-1], interleaved, x.device)
    c, s = scale * angles.cos(), scale * sign * angles.sin()
    y = x.clone()
    y[..., a] = x[..., a] * c - x[..., b] * s
    y[..., b] = x[..., b] * c + x[..., a] * s
    return y


def reach(x, half, interleaved, scale=1.0):
    """|a| + |b| of the pair that each channel belongs to, |x| where it belongs to none."""
    a, b = pairs(half, interleaved, x.device)
    m = x.abs().clone()
    m[..., a] = m[..., b] = (x[..., a].abs() + x[..., b].abs()) * max(scale, 1.0)
    return m


def norm64(x, w, eps):
    return x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + eps) * w


def angles64(positions, inv_freq):
    return positions.double()[..., None] * inv_freq.double()


def data(seed, *shape, dtype):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


SHAPES = [(1, 1, 1, 16, 16), (2, 17, 3, 32, 32), (1, 130, 24, 64, 64), (3, 33, 5, 64, 32), (2, 65, 7, 128, 128), (1, 40, 33, 128, 20),
          (2, 19, 4, 64, 2), (1, 700, 9, 16, 10), (1, 9, 260, 16, 8)]


@pytest.mark.parametrize("B,T,H,D,rot", SHAPES)
@pytest.mark.parametrize("interleaved,head_first", list(itertools.product([False, True], [False, True])))
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_rotary_and_its_gradient(B, T, H, D, rot, interleaved, head_first, dtype):
    scale = 1.25
    x = data(B * T + D, B, T, H, D, dtype=dtype)
    dy = data(B * T + D + 1, B, T, H, D, dtype=dtype)
    inv_freq, _ = fox.rotary_frequencies(rot, device="cuda")
    pos = torch.randint(0, 5000, (B, T), generator=torch.Generator().manual_seed(T)).cuda()
    lay = (lambda t: t.transpose(1, 2)) if head_first else (lambda t: t)
    xin = lay(x).detach().requires_grad_()
    y = fox.rotary_embedding(xin, inv_freq, pos, head_first=head_first, interleaved=interleaved, scale=scale)
    assert y.dtype == dtype and y.shape == xin.shape
    (dx,) = torch.autograd.grad(y, xin, lay(dy))
    a = angles64(pos, inv_freq)[:, :, None]
    for got, src, sign in ((y, x, 1.0), (dx, dy, -1.0)):
        ref = turn64(src.double(), a, interleaved, scale, sign)
        tol = half_step(dtype) * ref.abs() + 2 ** -20 * reach(src.double(), rot // 2, interleaved, scale) + tiny(dtype)
        err = (lay(got).double() - ref).abs()
        assert (err <= tol).all(), (err - tol).max().item()


@pytest.mark.parametrize("where", ["none", "int", "int32", "strided"])
def test_positions_in_every_form(where):
    x = data(3, 2, 50, 3, 64, dtype=torch.bfloat16)
    inv_freq, _ = fox.rotary_frequencies(64, device="cuda")
    given, at = {"none": (None, torch.arange(50)), "int": (1234567, 1234567 + torch.arange(50)),
                 "int32": (torch.arange(7, 57, dtype=torch.int32).cuda(), torch.arange(7, 57)),
                 "strided": (torch.arange(100, device="cuda")[::2], torch.arange(0, 100, 2))}[where]
    y = fox.rotary_embedding(x, inv_freq, given)
    ref = turn64(x.double(), angles64(at.cuda(), inv_freq)[:, None], False)
    tol = 2 ** -8 * ref.abs() + 2 ** -20 * reach(x.double(), 32, False)
    assert ((y.double() - ref).abs() <= tol).all()
    one = fox.rotary_embedding(x[1], inv_freq, given)       # a packed batch: three dimensions
    assert torch.equal(one, y[1])


@pytest.mark.parametrize("first", [-70000, 2 ** 20 + 1, 2 ** 31 - 40, 2 ** 40])
def test_angles_of_far_positions(first):
    """The product of position and frequency in 64 bits: its own rounding is 2^-53 of up to 2^40 radians, far below 2^-20 up to
    2^31; at 2^40 it is 2^-13 at the fastest frequency, which both sides share."""
    x = data(5, 1, 30, 2, 64, dtype=torch.float16)
    inv_freq, _ = fox.rotary_frequencies(64, device="cuda")
    y = fox.rotary_embedding(x, inv_freq, first)
    ref = turn64(x.double(), angles64(first + torch.arange(30, device="cuda"), inv_freq)[:, None], False)
    tol = 2 ** -11 * ref.abs() + 2 ** -20 * reach(x.double(), 32, False) + 2 ** -25
    assert ((y.double() - ref).abs() <= tol).all()


def test_strided_views_and_empty():
    """Slices of a projection's row, an expanded batch, a view that 16-byte loads cannot take, and no tokens."""
    inv_freq, _ = fox.rotary_frequencies(32, device="cuda")
    big = data(8, 2, 21, 9 * 64 + 3, dtype=torch.bfloat16)
    for x in (big[:, :, 64:4 * 64].view(2, 21, 3, 64), big[:, :, 3:3 + 3 * 64].view(2, 21, 3, 64),
              big[:1, :, :192].view(1, 21, 3, 64).expand(4, -1, -1, -1), big[:, ::2, :128].view(2, 11, 2, 64)):
        y = fox.rotary_embedding(x, inv_freq)
        assert torch.equal(y, fox.rotary_embedding(x.contiguous(), inv_freq))
    empty = big[:, :0, :128].view(2, 0, 2, 64).detach().requires_grad_()
    y = fox.rotary_embedding(empty, inv_freq)
    assert y.shape == empty.shape
    (dx,) = torch.autograd.grad(y, empty, torch.zeros_like(y))
    assert dx.shape == empty.shape


NORMS = [(1, 1, 1, 1, 16, 16), (2, 37, 4, 2, 32, 32), (1, 130, 24, 24, 64, 64), (2, 70, 6, 3, 64, 40), (1, 300, 16, 16, 128, 128),
         (3, 11, 33, 11, 128, 64), (1, 2100, 5, 5, 64, 12), (1, 5, 140, 70, 16, 4)]


@pytest.mark.parametrize("B,T,H,Hk,D,rot", NORMS)
@pytest.mark.parametrize("interleaved,shared", list(itertools.product([False, True], [False, True])))
@pytest.mark.parametrize("dtype,w_dtype", [(torch.bfloat16, torch.float32), (torch.float16, torch.float16),
                                           (torch.bfloat16, torch.bfloat16)])
def test_norm_rotary_and_its_gradients(B, T, H, Hk, D, rot, interleaved, shared, dtype, w_dtype):
    eps, scale = 1e-5, 1.1
    inv_freq, _ = fox.rotary_frequencies(rot, device="cuda")
    x = [data(T + i, B, T, h, D, dtype=dtype) for i, h in enumerate((H, Hk))]
    w = [(1 + 0.3 * data(T + 2 + i, D if shared else h * D, dtype=torch.float32)).to(w_dtype) for i, h in enumerate((H, Hk))]
    dy = [data(T + 4 + i, B, T, h, D, dtype=dtype) for i, h in enumerate((H, Hk))]
    leaves = [t.detach().requires_grad_() for t in (*x, *w)]
    out = fox.qk_norm_rotary(*leaves, inv_freq, 77, eps=eps, interleaved=interleaved, scale=scale)
    grads = torch.autograd.grad(out, leaves, dy)
    a = angles64(77 + torch.arange(T, device="cuda"), inv_freq)[:, None]
    parts = 600                                     # (at most: shares of the weights' gradients, 148 * 4)
    h16 = half_step(dtype)
    for i in range(2):
        x64, w64 = x[i].double(), w[i].double().view(-1, D)
        n = norm64(x64, w64, eps)
        ref = turn64(n, a, interleaved, scale)
        tol = h16 * ref.abs() + 2 ** -19 * reach(n, rot // 2, interleaved, scale) + tiny(dtype)
        assert ((out[i].double() - ref).abs() <= tol).all()
        dn = turn64(dy[i].double(), a, interleaved, scale, -1.0)
        m = reach(dy[i].double(), rot // 2, interleaved, scale)          # what dn's error is measured by
        r = torch.rsqrt(x64.pow(2).mean(-1, keepdim=True) + eps)
        xhat = x64 * r
        dx = r * (dn * w64 - xhat * (dn * w64 * xhat).mean(-1, keepdim=True))
        size = r * (m * w64.abs() + xhat.abs() * (m * w64 * xhat).abs().mean(-1, keepdim=True))
        assert grads[i].dtype == dtype
        # (dn 2^-20, r twice 2^-20, the products and the mean's sum of D terms 2^-20: 2^-18 of the terms' sizes)
        assert ((grads[i].double() - dx).abs() <= h16 * dx.abs() + 2 ** -18 * size + tiny(dtype)).all()
        axes = (0, 1, 2) if shared else (0, 1)
        heads = (H, Hk)[i]
        dw = (dn * xhat).sum(axes).flatten()
        terms = (m * xhat.abs()).sum(axes).flatten()
        chain = B * T + 16 if B * T < parts else B * T / 148 + 16        # of a thread, of the shares, of the last sums
        chain += parts / 16 * (heads if shared else 1) + 16
        tol = (2 ** -19 + chain * 2 ** -24) * terms
        if w_dtype != torch.float32:
            tol = tol + half_step(w_dtype) * dw.abs() + tiny(w_dtype)
        assert grads[2 + i].dtype == w_dtype and grads[2 + i].shape == w[i].shape
        assert ((grads[2 + i].double() - dw).abs() <= tol).all()


def test_norm_rotary_gradient_against_differences():
    """The gradients' products with a direction against central differences of the 64-bit formula.  The differences' own error
    is of third order (step 1e-4: below 1e-7 of the sum of sizes); the gradients' is their rounding, bounded as above."""
    B, T, H, Hk, D = 1, 24, 4, 2, 64
    inv_freq, _ = fox.rotary_frequencies(48, device="cuda")
    x = [data(i, B, T, h, D, dtype=torch.float16) for i, h in enumerate((H, Hk))]
    w = [1 + 0.2 * data(2 + i, h * D, dtype=torch.float32) for i, h in enumerate((H, Hk))]
    dy = [data(4 + i, B, T, h, D, dtype=torch.float16) for i, h in enumerate((H, Hk))]
    leaves = [t.detach().requires_grad_() for t in (*x, *w)]
    out = fox.qk_norm_rotary(*leaves, inv_freq, None)
    grads = torch.autograd.grad(out, leaves, dy)
    a = angles64(torch.arange(T, device="cuda"), inv_freq)[:, None]
    f = lambda i, xx, ww: (turn64(norm64(xx, ww.view(-1, D), 1e-5), a, False) * dy[i].double()).sum()
    for i in range(2):
        for k, (base, grad) in enumerate(((x[i].double(), grads[i]), (w[i].double(), grads[2 + i]))):
            d = data(9 + i, *base.shape, dtype=torch.float32).double()
            args = lambda t: (t, w[i].double()) if k == 0 else (x[i].double(), t)
            diff = (f(i, *args(base + 1e-4 * d)) - f(i, *args(base - 1e-4 * d))) / 2e-4
            off = (2 ** -11 if k == 0 else 2 ** -17) * (grad.double().abs() * d.abs()).sum() + 2 ** -16 * d.abs().sum()
            assert ((grad.double() * d).sum() - diff).abs() <= off


def test_one_result_unused_and_frozen_inputs():
    inv_freq, _ = fox.rotary_frequencies(64, device="cuda")
    q, k = [data(i, 2, 9, 3, 64, dtype=torch.bfloat16).requires_grad_() for i in range(2)]
    w = torch.ones(64, device="cuda")
    out = fox.qk_norm_rotary(q, k, w, w, inv_freq)
    dq, dk = torch.autograd.grad(out[0].float().sum(), [q, k], retain_graph=True)
    assert dk.abs().max() == 0 and dq.abs().max() > 0
    with torch.no_grad():
        assert not fox.qk_norm_rotary(q, k, w, w, inv_freq)[0].requires_grad
    frozen = fox.qk_norm_rotary(q.detach(), k, w, w, inv_freq)
    (dk2,) = torch.autograd.grad(frozen[1].float().sum(), [k])
    assert dk2.abs().max() > 0
    torch.autograd.grad(out[1].float().sum(), [k])
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(out[1].float().sum(), [k])


def test_inference_mode_and_the_traced_functions():
    """Under inference_mode, and by the autograd functions that torch.jit.trace records: the same bits, gradients too."""
    inv_freq, _ = fox.rotary_frequencies(64, device="cuda")
    q, k = [data(i, 2, 13, 3, 64, dtype=torch.float16) for i in range(2)]
    w = torch.rand(192, device="cuda") + 0.5
    with torch.inference_mode():
        a = [fox.rotary_embedding(q, inv_freq, 5), *fox.qk_norm_rotary(q, k, w, w, inv_freq, 5)]
    pos = 5 + torch.arange(13, device="cuda")
    f = lambda q, k, w: [fox.rotary_embedding(q, inv_freq, pos), *fox.qk_norm_rotary(q, k, w, w, inv_freq, pos)]
    traced = torch.jit.trace(f, (q, k, w), check_trace=False)
    for x, y in zip(a, traced(q, k, w)):
        assert torch.equal(x, y)
    leaves = [t.clone().requires_grad_() for t in (q, k, w)]
    dy = [data(7 + i, 2, 13, 3, 64, dtype=torch.float16) for i in range(3)]
    from forgetting_transformer_b200 import rotary
    args = (inv_freq, pos, False, False, 1.0)
    by_class = [rotary._Rotate.apply(leaves[0], *args), *rotary._NormRotate.apply(leaves[0], leaves[1], leaves[2], leaves[2], inv_freq, pos, 1e-5, False, False, 1.0)]
    got = torch.autograd.grad(by_class, leaves, dy)
    want = torch.autograd.grad(f(*leaves), leaves, dy)
    for x, y in zip(got, want):
        assert torch.equal(x, y)


def test_streams_and_graphs():
    """On a stream of the caller's, forward and backward captured in a graph and replayed on new values."""
    inv_freq, _ = fox.rotary_frequencies(64, device="cuda")
    q, k = [data(i, 1, 40, 4, 64, dtype=torch.bfloat16).requires_grad_() for i in range(2)]
    w = [torch.ones(256, device="cuda").requires_grad_() for _ in range(2)]
    pos = torch.zeros(40, dtype=torch.int32, device="cuda")
    dy = [data(5 + i, 1, 40, 4, 64, dtype=torch.bfloat16) for i in range(2)]

    def step():
        out = fox.qk_norm_rotary(q, k, *w, inv_freq, pos)
        return [*out, *torch.autograd.grad(out, [q, k, *w], dy)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            got = step()
        with torch.no_grad():
            q.copy_(data(11, 1, 40, 4, 64, dtype=torch.bfloat16))
            pos.copy_(torch.arange(100, 140))
        g.replay()
        want = step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("scaling", [dict(scaling="linear", factor=4.0), dict(scaling="ntk", factor=4.0),
                                     dict(scaling="yarn", factor=8.0, original_length=2048)])
def test_rotary_module(scaling):
    """The module's two ways, in a layer's type, with scaled frequencies; norms in front."""
    m = fox.RotaryEmbedding(64, 500000.0, **scaling).cuda().bfloat16()
    q, k = [data(i, 1, 30, 2, 64, dtype=torch.bfloat16) for i in range(2)]
    f, s = fox.rotary_frequencies(64, 500000.0, **scaling)
    assert f.dtype == torch.float32 and m.scale == s
    a = angles64(5000 + torch.arange(30, device="cuda"), f.cuda())[:, None]
    for got, x in zip(m(q, k, 5000), (q, k)):
        ref = turn64(x.double(), a, False, s)
        assert ((got.double() - ref).abs() <= 2 ** -8 * ref.abs() + 2 ** -20 * reach(x.double(), 32, False, s)).all()
    w = torch.full((64,), 0.5, device="cuda")
    for got, x in zip(m.norm(q, k, w, w, 5000), (q, k)):
        n = norm64(x.double(), 0.5, 1e-5)
        ref = turn64(n, a, False, s)
        assert ((got.double() - ref).abs() <= 2 ** -8 * ref.abs() + 2 ** -19 * reach(n, 32, False, s)).all()


def composed(layer, x, cache=None, layer_idx=0):
    """The attention layer from its modules and the public operators, as its documentation has it."""
    B, T, C = x.shape
    H, D = layer.num_heads, layer.head_dim
    past = cache.get_seq_length(layer_idx) if cache is not None else 0
    k_state, v_state = (cache.key_shift_cache[layer_idx], cache.value_shift_cache[layer_idx]) if cache is not None else (None, None)
    q, k, v = layer.q_proj(x), layer.k_proj(x, None, k_state), layer.v_proj(x, None, v_state)
    q, k = layer.rotary.norm(q.view(B, T, H, D), k.view(B, T, H, D), layer.q_norm.weight, layer.k_norm.weight, past, eps=layer.q_norm.eps)
    q, k, v = [t.reshape(B, T, H, D).transpose(1, 2) for t in (q, k, v)]
    logit = layer.fgate_proj(x).transpose(1, 2)
    if cache is None:
        o = fox.forgetting_attention_from_gate_logits(q, k, v, logit, head_first=True, sm_scale=D ** -0.5)
    else:
        k, v, g = cache.update(k, v, torch.nn.functional.logsigmoid(logit.float()), layer_idx)
        o = fox.forgetting_attention(q, k, v, g, head_first=True, sm_scale=D ** -0.5)
    return layer.o_proj(layer.output_norm(o.transpose(1, 2).reshape(B, T, C), layer.ogate_proj(x)))


def test_layer_with_rotary_positions():
    """The layer with rotary positions is its modules with ``RotaryEmbedding.norm`` in the norms' place: the same calls, so the
    same bits, forward, backward and with a cache; a block with such a layer does not take the native path, which has none."""
    torch.manual_seed(0)
    block = fox.FoxProBlock(256, 4, 512, rotary=fox.RotaryEmbedding(64, 10000.0)).cuda().bfloat16()
    plain = fox.FoxProBlock(256, 4, 512).cuda().bfloat16()
    plain.load_state_dict(block.state_dict())
    x = data(1, 2, 37, 256, dtype=torch.bfloat16)
    layer = block.attn
    grads = []
    for f in (lambda y: layer(y), lambda y: composed(layer, y)):
        layer.zero_grad()
        xin = x.clone().requires_grad_()
        out = f(xin)
        out.backward(data(2, *out.shape, dtype=torch.bfloat16))
        grads.append([out.detach(), xin.grad] + [p.grad.clone() for p in layer.parameters()])
    for a, b in zip(*grads):
        assert torch.equal(a, b)
    with torch.no_grad():
        out = block(x)
        h, res = block.mlp_norm(layer(block.attn_norm(x)), x, True)
        assert torch.equal(out, res + block.mlp(h))
        assert not torch.equal(out, plain(x))
        caches = []
        for f in (layer, composed):
            cache = fox.FgateCache(64)
            s = layer.init_shift_state(2)
            cache.update_shift_cache(s["key_shift"], s["value_shift"], 0)
            call = (lambda y: layer(y, None, cache, 0)) if f is layer else (lambda y: composed(layer, y, cache))
            caches.append([call(x[:, :30])] + [call(x[:, t:t + 1]) for t in range(30, 37)])
        for a, b in zip(*caches):
            assert torch.equal(a, b)


def test_module_trains_after_inference():
    """Frequencies that came to the device under inference mode serve a backward pass afterwards."""
    m = fox.RotaryEmbedding(32)
    q, k = [data(i, 1, 9, 2, 64, dtype=torch.bfloat16) for i in range(2)]
    with torch.inference_mode():
        first = m(q, k, 3)
    leaf = q.clone().requires_grad_()
    out = m(leaf, k, 3)
    assert torch.equal(out[0], first[0]) and torch.equal(out[1], first[1])
    out[0].backward(torch.ones_like(leaf))
    assert leaf.grad.abs().max() > 0


def test_layer_with_scale_prunes_within_its_tolerance(monkeypatch):
    """The closed-form threshold counts the rotation's scale, by which both q and k are longer: -(2 bound + ln T) + tolerance with
    bound = scale^2 max|w_q| max|w_k| sqrt(D) (here 1 x 1 x 8)."""
    from forgetting_transformer_b200 import block as block_module
    rot = fox.RotaryEmbedding(64, scaling="yarn", factor=16.0, original_length=2048)
    layer = fox.FoxProAttentionLayer(128, 2, log_pruning_tolerance=-10.0, rotary=rot).cuda().bfloat16()
    seen = []
    inner = block_module.forgetting_attention_from_gate_logits
    monkeypatch.setattr(block_module, "forgetting_attention_from_gate_logits",
                        lambda *a, **k: seen.append(k["adaptive_threshold"]) or inner(*a, **k))
    with torch.no_grad():
        layer(data(1, 1, 128, 128, dtype=torch.bfloat16))
    want = -(2 * rot.scale ** 2 * 8 + math.log(128)) - 10
    # the weights are 1 in bf16; scale^2, bound, sum and result are rounded to bf16: 4 x 2^-8, of terms up to |want|
    assert rot.scale > 1.2 and (seen[0].double() - want).abs().max() <= 4 * 2 ** -8 * abs(want)


def test_layer_calls_norms_that_are_not_its_own():
    """Replaced norms of q and k, and those with hooks, are called; the rotation follows them."""
    layer = fox.FoxProAttentionLayer(128, 2, rotary=fox.RotaryEmbedding(64)).cuda().bfloat16()
    x = data(1, 1, 20, 128, dtype=torch.bfloat16)
    calls = []

    class Half(torch.nn.Module):
        def forward(self, x):
            calls.append("half")
            return x / 2
    with torch.no_grad():
        fused = layer(x)
        handle = layer.q_norm.register_forward_hook(lambda *a: calls.append("hook"))
        hooked = layer(x)
        handle.remove()
        assert calls == ["hook"] and torch.equal(layer(x), fused) and calls == ["hook"]
        norms = [fox.GroupNorm(2, 128, is_rms_norm=True).cuda().bfloat16() for _ in range(2)]
        layer.rotary.norm = lambda q, k, w_q, w_k, past, eps: layer.rotary(
            *[n(x.flatten(2)).view(x.shape) for n, x in zip(norms, (q, k))], past)
        assert torch.equal(hooked, composed(layer, x))
        del layer.rotary.norm
        layer.q_norm = layer.k_norm = Half()
        assert not torch.equal(layer(x), fused) and calls == ["hook", "half", "half"]


def test_second_derivatives():
    """The rotation's gradient is the rotation back, and that one's the rotation: |y|^2 / 2 has the gradient x (scale 1) and the second
    derivative v along v, each value rounded twice.  The norms' second derivative is refused, not zero."""
    inv_freq, _ = fox.rotary_frequencies(64, device="cuda")
    x = data(1, 1, 9, 2, 64, dtype=torch.bfloat16).requires_grad_()
    v = data(2, 1, 9, 2, 64, dtype=torch.bfloat16)
    y = fox.rotary_embedding(x, inv_freq, 7)
    (g,) = torch.autograd.grad((y * y).sum() / 2, [x], create_graph=True)
    (h,) = torch.autograd.grad(g, [x], v)
    for got, ref in ((g, x), (h, v)):
        # the first rounding's half steps, turned, are 2^-8 of the turned pair's |a| + |b| at most, which is 2^0.5 of the pair's own
        slack = (2 ** 0.5 * 2 ** -8 + 2 ** -19) * reach(ref.double(), 32, False)
        assert ((got.double() - ref.double()).abs() <= 2 ** -8 * (ref.double().abs() + slack) + slack + 2 ** -7 * slack).all()
    q, k = [data(i, 1, 9, 2, 64, dtype=torch.bfloat16).requires_grad_() for i in range(2)]
    w = torch.ones(64, device="cuda")
    out = fox.qk_norm_rotary(q, k, w, w, inv_freq)
    g = torch.autograd.grad(out[0].float().pow(2).sum(), [q], create_graph=True)
    with pytest.raises(RuntimeError, match="no second derivative"):
        torch.autograd.grad(g[0].float().sum(), [q])
    out = fox.qk_norm_rotary(q, k, w, w, inv_freq)
    assert not torch.autograd.grad(out[0].float().sum(), [q])[0].requires_grad


@pytest.mark.parametrize("T,H,D", [(120001, 3, 16), (30011, 32, 64)])
def test_many_tokens(T, H, D):
    """Several ranges of tokens for every place of a CTA on the GPU, the last of them short: every token is turned, and normed, once."""
    x = data(T, 1, T, H, D, dtype=torch.bfloat16)
    inv_freq, _ = fox.rotary_frequencies(D, device="cuda")
    a = angles64(torch.arange(T, device="cuda"), inv_freq)[None, :, None]
    w = torch.full((D,), 0.75, device="cuda")
    y = fox.rotary_embedding(x, inv_freq)
    q, k = fox.qk_norm_rotary(x, x, w, w, inv_freq)
    n = norm64(x.double(), 0.75, 1e-5)
    for got, src, slack in ((y, x.double(), 2 ** -20), (q, n, 2 ** -19), (k, n, 2 ** -19)):
        ref = turn64(src, a, False)
        assert ((got.double() - ref).abs() <= 2 ** -8 * ref.abs() + slack * reach(src, D // 2, False)).all()


def test_module_in_a_capture():
    """A module whose frequencies are not yet on the device refuses to be captured, without harm to the capture; one that has been
    called, or asked for them, is replayed on new values."""
    m = fox.RotaryEmbedding(64)
    q, k = [data(i, 1, 9, 2, 64, dtype=torch.bfloat16) for i in range(2)]
    stays = torch.zeros(4, device="cuda")
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        with pytest.raises(fox.FoxError, match="once before"):
            m(q, k, 5)
        stays.add_(1)
    g.replay()
    assert stays.tolist() == [1.0] * 4
    m.inv_freq(q.device)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = m(q, k, 5)
    q.copy_(data(3, 1, 9, 2, 64, dtype=torch.bfloat16))
    g.replay()
    for a, b in zip(got, m(q, k, 5)):
        assert torch.equal(a, b)


def big(seed, *shape, dtype):
    return torch.randn(*shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").to(dtype)


def several_tiles(kind, B, T, heads, D, rot, interleaved):
    """Whether a CTA's range of tokens is longer than the tile whose angles it holds, so that it comes to a second one; and, with
    sequences that are no multiple of the range, crosses from one into the next."""
    from forgetting_transformer_b200 import _lib
    per = _lib.load().fox_rotary_range(kind, B, T, heads, D, rot // 2, interleaved)
    return per > (16 if not interleaved and rot // 2 % 4 else 32) and T % per


@pytest.mark.parametrize("T,H,D,rot,interleaved,head_first,dtype", [
    (25603, 16, 128, 128, False, False, torch.bfloat16), (25603, 32, 64, 64, True, False, torch.float16),
    (25603, 32, 64, 32, False, True, torch.float16), (25603, 128, 16, 12, True, False, torch.bfloat16),
    (25603, 64, 32, 32, False, False, torch.bfloat16), (4001, 16, 128, 44, False, False, torch.bfloat16),
    (4001, 16, 128, 42, False, True, torch.float16), (8001, 16, 64, 22, False, False, torch.float16),
    (8001, 64, 16, 12, False, False, torch.bfloat16)])
def test_rotary_of_ranges_in_several_tiles(T, H, D, rot, interleaved, head_first, dtype):
    """Ranges of more tokens than a tile, across sequences with positions of their own; the gradient is the same kernel."""
    B = 3
    assert several_tiles(0, B, T, H, D, rot, interleaved)
    inv_freq, _ = fox.rotary_frequencies(rot, device="cuda")
    pos = torch.randint(0, 50000, (B, T), generator=torch.Generator().manual_seed(T)).int().cuda()
    lay = (lambda t: t.transpose(1, 2)) if head_first else (lambda t: t)
    x, dy = [lay(big(T + i, *((B, H, T, D) if head_first else (B, T, H, D)), dtype=dtype)) for i in range(2)]
    xin = lay(x).detach().requires_grad_()
    y = fox.rotary_embedding(xin, inv_freq, pos, head_first=head_first, interleaved=interleaved)
    (dx,) = torch.autograd.grad(y, xin, lay(dy))
    for b in range(B):
        a = angles64(pos[b], inv_freq)[:, None]
        for got, src, sign in ((y, x, 1.0), (dx, dy, -1.0)):
            src = src[b].double()
            ref = turn64(src, a, interleaved, 1.0, sign)
            tol = half_step(dtype) * ref.abs() + 2 ** -20 * reach(src, rot // 2, interleaved) + tiny(dtype)
            assert ((lay(got)[b].double() - ref).abs() <= tol).all()


@pytest.mark.parametrize("T,H,Hk,D,rot,interleaved,shared,dtype", [
    (25603, 8, 8, 128, 128, False, False, torch.bfloat16), (25603, 12, 4, 128, 64, True, True, torch.float16),
    (6001, 16, 16, 128, 128, False, False, torch.bfloat16), (6001, 16, 16, 128, 128, True, True, torch.bfloat16),
    (6001, 16, 16, 128, 44, False, True, torch.float16), (6001, 16, 16, 128, 42, False, False, torch.bfloat16),
    (8003, 12, 4, 64, 64, False, True, torch.float16), (8003, 12, 4, 64, 22, False, False, torch.bfloat16),
    (10007, 24, 24, 16, 16, False, False, torch.bfloat16), (10007, 40, 8, 32, 24, True, True, torch.bfloat16)])
def test_norm_rotary_of_ranges_in_several_tiles(T, H, Hk, D, rot, interleaved, shared, dtype):
    """As above for the norms, whose backward carries the weights' gradients from tile to tile.  dw: every addition of a thread's
    tokens, of a CTA's heads where they share a weight, and of the shares (32 groups, then those) rounds what has been added so
    far by 2^-24; each term is off by 2^-19 of its size."""
    from forgetting_transformer_b200 import _lib
    B, eps = 3, 1e-5
    assert several_tiles(2, B, T, H + Hk, D, rot, interleaved) and (T < 25603 or several_tiles(1, B, T, H + Hk, D, rot, interleaved))
    inv_freq, _ = fox.rotary_frequencies(rot, device="cuda")
    pos = torch.randint(0, 50000, (B, T), generator=torch.Generator().manual_seed(T)).int().cuda()
    x = [big(T + i, B, T, h, D, dtype=dtype) for i, h in enumerate((H, Hk))]
    dy = [big(T + 2 + i, B, T, h, D, dtype=dtype) for i, h in enumerate((H, Hk))]
    w = [1 + 0.3 * data(T + 4 + i, D if shared else h * D, dtype=torch.float32) for i, h in enumerate((H, Hk))]
    leaves = [t.detach().requires_grad_() for t in (*x, *w)]
    out = fox.qk_norm_rotary(*leaves, inv_freq, pos, eps=eps, interleaved=interleaved)
    grads = torch.autograd.grad(out, leaves, dy)
    h16 = half_step(dtype)
    ranges = _lib.load().fox_qk_norm_rotary_partials(B, T, H, Hk, D)
    for i, heads in enumerate((H, Hk)):
        w64 = w[i].double().view(-1, D)
        dw = terms = 0
        for b in range(B):
            a = angles64(pos[b], inv_freq)[:, None]
            x64, dy64 = x[i][b].double(), dy[i][b].double()
            r = torch.rsqrt(x64.pow(2).mean(-1, keepdim=True) + eps)
            xhat = x64 * r
            n = xhat * w64
            ref = turn64(n, a, interleaved)
            assert ((out[i][b].double() - ref).abs() <= h16 * ref.abs() + 2 ** -19 * reach(n, rot // 2, interleaved) + tiny(dtype)).all()
            dn, m = turn64(dy64, a, interleaved, 1.0, -1.0), reach(dy64, rot // 2, interleaved)
            dx = r * (dn * w64 - xhat * (dn * w64 * xhat).mean(-1, keepdim=True))
            size = r * (m * w64.abs() + xhat.abs() * (m * w64 * xhat).abs().mean(-1, keepdim=True))
            assert ((grads[i][b].double() - dx).abs() <= h16 * dx.abs() + 2 ** -18 * size + tiny(dtype)).all()
            axes = (0, 1) if shared else (0,)
            dw, terms = dw + (dn * xhat).sum(axes).flatten(), terms + (m * xhat.abs()).sum(axes).flatten()
        over = H + Hk if shared else 1
        chain = -(-B * T // ranges) + over + -(-ranges // 32) * over + 32
        assert ((grads[2 + i].double() - dw).abs() <= (2 ** -19 + chain * 2 ** -24) * terms).all()
