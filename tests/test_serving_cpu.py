"""Refusals of the rotary and paged-cache operators, which come before anything runs on a GPU, and the frequencies."""
import copy
import math
import pickle

import pytest
import torch
import torch.autograd.forward_ad as fwAD

import forgetting_transformer_b200 as fox
from forgetting_transformer_b200 import _lib


def bf(*shape):
    return torch.zeros(*shape, dtype=torch.bfloat16)


F32 = torch.ones(32)


@pytest.mark.parametrize("call,why", [
    (lambda: fox.rotary_embedding(torch.zeros(1, 4, 2, 64), F32), "Only torch.float16"),
    (lambda: fox.rotary_embedding(bf(4, 64), F32), "3 or 4 dimensions"),
    (lambda: fox.rotary_embedding(bf(1, 4, 2, 48), F32), "head dims"),
    (lambda: fox.rotary_embedding(bf(1, 4, 2, 32), F32), "inv_freq must have"),
    (lambda: fox.rotary_embedding(bf(1, 4, 2, 64), F32[:0]), "inv_freq must have"),
    (lambda: fox.rotary_embedding(bf(1, 4, 2, 64), F32.double()), "torch.float32"),
    (lambda: fox.rotary_embedding(bf(1, 4, 2, 64), F32, torch.zeros(5, dtype=torch.int32)), "positions must have the shape"),
    (lambda: fox.rotary_embedding(bf(2, 4, 2, 64), F32, torch.zeros(3, 4, dtype=torch.int32)), "positions must have the shape"),
    (lambda: fox.rotary_embedding(bf(1, 4, 2, 64), F32, torch.zeros(4)), "torch.int32 or torch.int64"),
    (lambda: fox.rotary_embedding(bf(1, 4, 2, 64), F32, 1.5), "integer"),
    (lambda: fox.qk_norm_rotary(bf(1, 4, 2, 64), bf(1, 5, 2, 64), F32, F32, F32), "agree"),
    (lambda: fox.qk_norm_rotary(bf(1, 4, 2, 64), bf(1, 4, 2, 64).half(), F32, F32, F32), "agree"),
    (lambda: fox.qk_norm_rotary(bf(1, 4, 2, 64), bf(1, 4, 2, 64), torch.ones(32), torch.ones(64), F32), "q_weight"),
    (lambda: fox.qk_norm_rotary(bf(1, 4, 2, 64), bf(1, 4, 2, 64), torch.ones(64), torch.ones(64).int(), F32), "k_weight"),
])
def test_rotary_refusals(call, why):
    with pytest.raises(AssertionError, match=why):
        call()


def test_no_cpu_path():
    i = lambda *s: torch.zeros(*s, dtype=torch.int32)
    with pytest.raises(_lib.FoxError, match="no CPU path"):
        fox.rotary_embedding(bf(1, 4, 2, 64), F32)
    with pytest.raises(_lib.FoxError, match="no CPU path"):
        fox.qk_norm_rotary(bf(1, 4, 2, 64), bf(1, 4, 2, 64), torch.ones(64), torch.ones(128), F32)
    with pytest.raises(_lib.FoxError, match="no CPU path"):
        fox.page_tables(i(2), i(2), i(2, 3), i(5), i(1), 16, 4)
    with pytest.raises(_lib.FoxError, match="no CPU path"):
        fox.release_pages(i(2), i(2), i(2, 3), i(5), i(1), 16)
    pool = pages()
    with pytest.raises(_lib.FoxError, match="no CPU path"):
        fox.paged_update(*pool, bf(4, 2, 64), bf(4, 2, 64), torch.zeros(4, 2), i(4))
    with pytest.raises(_lib.FoxError, match="no CPU path"):
        fox.paged_forgetting_attention(bf(3, 2, 64), *pool, i(3, 4), i(3))


def test_frequencies_have_no_gradient():
    f = F32.clone().requires_grad_()
    with pytest.raises(_lib.FoxError, match="no gradient for inv_freq"):
        fox.rotary_embedding(bf(1, 4, 2, 64), f)
    with pytest.raises(_lib.FoxError, match="no gradient for inv_freq"):
        fox.qk_norm_rotary(bf(1, 4, 2, 64), bf(1, 4, 2, 64), torch.ones(64), torch.ones(64), f)
    with torch.no_grad(), pytest.raises(_lib.FoxError, match="no CPU path"):
        fox.rotary_embedding(bf(1, 4, 2, 64), f)


def pages(P=5, Hk=2, H=2, page=16, D=64, dtype=torch.bfloat16):
    return (torch.zeros(P, Hk, page, D, dtype=dtype), torch.zeros(P, Hk, page, D, dtype=dtype), torch.zeros(P, H, page))


@pytest.mark.parametrize("change,why", [
    (dict(page=24), "power of two"), (dict(page=8), "power of two"), (dict(D=48), "head dims"), (dict(H=3), "multiple"),
    (dict(dtype=torch.float32), "float16"),
])
def test_pool_refusals(change, why):
    kw = dict(P=5, Hk=2, H=2, page=16, D=64, dtype=torch.bfloat16, **{})
    kw.update(change)
    with pytest.raises(AssertionError, match=why):
        fox.paged_forgetting_attention(bf(3, kw["H"], kw["D"]), *pages(**kw), torch.zeros(3, 4, dtype=torch.int32),
                                       torch.zeros(3, dtype=torch.int32))


def test_paged_refusals():
    i = lambda *s: torch.zeros(*s, dtype=torch.int32)
    k, v, g = pages()
    att = fox.paged_forgetting_attention
    for args, why in [((bf(3, 2, 32), k, v, g, i(3, 4), i(3)), "head dim"), ((bf(3, 1, 64), k, v, g, i(3, 4), i(3)), "heads"),
                      ((bf(3, 2, 64).half(), k, v, g, i(3, 4), i(3)), "type"), ((bf(3, 2, 64), k, v, g, i(2, 4), i(3)), "request"),
                      ((bf(3, 2, 64), k, v, g, i(3, 4).long(), i(3)), "int32"), ((bf(3, 2, 64), k, v, g, i(4, 3).t(), i(3)), "contiguous"),
                      ((bf(3, 2, 64), k, v[:4], g, i(3, 4), i(3)), "equal shapes"), ((bf(3, 2, 64), k, v, g[:4], i(3, 4), i(3)), "gate_pages"),
                      ((bf(3, 2, 64), k, v, g.double(), i(3, 4), i(3)), "float32"),
                      ((bf(3, 2, 64), k, v, torch.zeros(5, 2, 17)[:, :, 1:], i(3, 4), i(3)), "16 bytes"),
                      ((bf(3, 2, 64), torch.zeros(5, 2, 16, 68, dtype=torch.bfloat16)[..., 4:], v, g, i(3, 4), i(3)), "16 bytes"),
                      ((bf(3, 2, 64), k.transpose(2, 3).contiguous().transpose(2, 3), v, g, i(3, 4), i(3)), "contiguous")]:
        with pytest.raises(AssertionError, match=why):
            att(*args)
    with pytest.raises(_lib.FoxError, match="no gradients"):
        att(bf(3, 2, 64).requires_grad_(), k, v, g, i(3, 4), i(3))
    up = fox.paged_update
    for args, why in [((k, v, g, bf(4, 3, 64), bf(4, 3, 64), torch.zeros(4, 2), i(4)), "heads"),
                      ((k, v, g, bf(4, 2, 64), bf(3, 2, 64), torch.zeros(4, 2), i(4)), "heads"),
                      ((k, v, g, bf(4, 2, 64).half(), bf(4, 2, 64), torch.zeros(4, 2), i(4)), "type"),
                      ((k, v, g, bf(4, 2, 64), bf(4, 2, 64), torch.zeros(4, 3), i(4)), "gates"),
                      ((k, v, g, bf(4, 2, 64), bf(4, 2, 64), bf(4, 2), i(4)), "float32"),
                      ((k, v, g, bf(4, 2, 64), bf(4, 2, 64), torch.zeros(4, 2), i(5)), "slots"),
                      ((k, v, g, bf(4, 2, 64), bf(4, 2, 64), torch.zeros(4, 2), torch.zeros(4)), "slots")]:
        with pytest.raises(AssertionError, match=why):
            up(*args)
    with pytest.raises(_lib.FoxError, match="no gradients"):
        up(k, v, g, bf(4, 2, 64).requires_grad_(), bf(4, 2, 64), torch.zeros(4, 2), i(4))
    tab = fox.page_tables
    for args, why in [((i(2), i(3), i(2, 3), i(5), i(1), 16, 4), "each request"), ((i(2), i(2), i(2, 3), i(5), i(2), 16, 4), "num_free"),
                      ((i(2).long(), i(2), i(2, 3), i(5), i(1), 16, 4), "int32"), ((i(2), i(2), i(2, 3), i(5), i(1), 20, 4), "power of two"),
                      ((i(2), i(2), i(2, 3), i(5), i(1), 16, -1), "max_tokens"), ((i(0), i(0), i(0, 3), i(5), i(1), 16, 4), "one at least"),
                      ((i(2), i(2), i(1, 3).expand(2, 3), i(5), i(1), 16, 4), "overlap")]:
        with pytest.raises(AssertionError, match=why):
            tab(*args)
    with pytest.raises(AssertionError, match="keep"):
        fox.release_pages(i(2), i(3), i(2, 3), i(5), i(1), 16)


def test_cache_refusals():
    ok = dict(num_layers=1, num_pages=4, page_size=16, num_heads=4, head_dim=64, max_requests=2, max_length=40, device="cpu")
    c = fox.PagedFgateCache(**ok)
    assert c.block_table.shape == (2, 3) and c.free_pages.tolist() == [3, 2, 1, 0] and c.num_free.tolist() == [4] and len(c) == 1
    for bad in (dict(page_size=24), dict(num_kv_heads=3), dict(num_pages=0), dict(max_length=0)):
        with pytest.raises(ValueError):
            fox.PagedFgateCache(**{**ok, **bad})


def test_c_interface_refuses_sizes():
    """Bad sizes come back as codes, before any device is touched (there is none here)."""
    lib = _lib.load()
    t, a = _lib.Tensor4(16, 8, 8, 8), 16
    rot = lambda **c: lib.fox_rotary(*{**dict(dev=0, st=None, dt=1, B=1, T=1, H=1, D=64, x=t, f=a, half=32, inter=0, scale=1.0, inv=0, pos=None,
                                             p64=0, sb=0, stt=0, first=0, y=t), **c}.values())
    assert rot(D=48) == -2 and rot(half=33) == -1 and rot(half=0) == -1 and rot(B=0) == -1 and rot(dt=2) == -1
    assert rot(T=2 ** 31) == -8 and rot(B=2 ** 20, T=2 ** 12) == -8 and rot(x=_lib.Tensor4(8, 8, 8, 8)) == -3 and rot(f=None) == -1
    att = lambda **c: lib.fox_paged_attn(*{**dict(dev=0, st=None, dt=1, R=1, H=4, Hk=2, D=64, P=4, page=16, w=2, q=a, qr=8, qh=8, k=t, v=t, g=a, gp=4,
                                                 gh=4, tab=a, ld=2, len=a, sc=1.0, o=a, orr=8, oh=8, L=None, ws=a, status=a), **c}.values())
    assert att(D=8) == -2 and att(H=3) == -1 and att(page=17) == -1 and att(ld=1) == -1 and att(P=2 ** 28) == -8 and att(gp=2) == -3
    assert att(R=0) == -1 and att(q=8) == -3 and att(ws=None) == -1 and att(status=None) == -1
    assert att(H=64, Hk=64, page=65536, w=2 ** 15, ld=2 ** 15) == -8     # more than 2^30 tiles in one request
    assert lib.fox_paged_attn_workspace_floats(0, 1, 1, 64) == 1 and lib.fox_qk_norm_rotary_partials(0, 0, 0, 0, 0) == 1


def test_frequencies():
    f, s = fox.rotary_frequencies(64)
    assert s == 1.0 and f.dtype == torch.float32 and f.shape == (32,)
    want = torch.tensor([10000.0 ** (-2 * i / 64) for i in range(32)], dtype=torch.float64)
    assert ((f.double() - want).abs() <= 2 ** -24 * want).all()
    lin, _ = fox.rotary_frequencies(64, scaling="linear", factor=4.0)
    assert ((lin.double() * 4 - want).abs() <= 2 ** -24 * want).all()
    ntk, _ = fox.rotary_frequencies(64, scaling="ntk", factor=4.0)
    assert ntk[0] == 1 and abs(float(ntk[-1]) * 4 / float(want[-1]) - 1) < 2 ** -22
    yarn, s = fox.rotary_frequencies(64, scaling="yarn", factor=8.0, original_length=4096)
    assert s == pytest.approx(0.1 * math.log(8) + 1)
    turns = 4096 * want / (2 * math.pi)
    assert torch.equal(yarn[turns > 32], f[turns > 32])
    slow = turns < 1
    assert slow.any() and ((yarn[slow].double() * 8 - want[slow]).abs() <= 2 ** -24 * want[slow]).all()
    assert (yarn[:-1] > yarn[1:]).all()
    for bad in (dict(dim=63), dict(dim=0), dict(dim=64, scaling="yarn", factor=2.0), dict(dim=64, scaling="other"),
                dict(dim=64, factor=0.0), dict(dim=2, scaling="ntk", factor=2.0)):
        with pytest.raises(ValueError):
            fox.rotary_frequencies(**bad)


def test_module_keeps_its_frequencies():
    """Built on the meta device or under inference mode, copied and pickled: the frequencies are the arguments' own, on any device
    asked for, and no copy of one device goes with the module to another."""
    want, _ = fox.rotary_frequencies(64, 500000.0)
    cpu = torch.device("cpu")
    with torch.device("meta"):
        meta = fox.RotaryEmbedding(64, 500000.0)
        assert fox.rotary_frequencies(64)[0].is_meta
    with torch.inference_mode():
        made = fox.RotaryEmbedding(64, 500000.0)
        assert not made.inv_freq(cpu).is_inference()
    used = fox.RotaryEmbedding(64, 500000.0)
    used.inv_freq(cpu)
    for m in (meta, made, used, copy.deepcopy(used), pickle.loads(pickle.dumps(used))):
        assert torch.equal(m.inv_freq(cpu), want)
    assert used._on_device and not pickle.loads(pickle.dumps(used))._on_device


def test_no_heads_are_refused():
    with pytest.raises(AssertionError, match="one head"):
        fox.qk_norm_rotary(bf(1, 4, 0, 64), bf(1, 4, 2, 64), torch.ones(64), torch.ones(64), F32)
    with pytest.raises(AssertionError, match="one head"):
        fox.qk_norm_rotary(bf(1, 4, 2, 64), bf(1, 4, 0, 64), torch.ones(64), torch.ones(64), F32)


def test_one_request_out_of_many_columns():
    """Vectors of one element may carry any stride: they pass the checks that come before the device's."""
    state = torch.zeros(1, 3, dtype=torch.int32)
    i = lambda *s: torch.zeros(*s, dtype=torch.int32)
    assert state[:, 1].stride(0) == 3
    with pytest.raises(_lib.FoxError, match="no CPU path"):
        fox.page_tables(state[:, 0], state[:, 1], i(1, 3), i(5), state[:, 2], 16, 4)
    with pytest.raises(AssertionError, match="contiguous"):
        fox.page_tables(i(2, 3)[:, 0], i(2), i(2, 3), i(5), i(1), 16, 4)


def paged_calls():
    """Each paged operator on valid arguments, as a function of those of them that may carry values: (name, function, inputs)."""
    i = lambda *s: torch.zeros(*s, dtype=torch.int32)
    k, v, g = pages()
    q, rows, gates = bf(3, 2, 64), bf(4, 2, 64), torch.zeros(4, 2)
    return [("page_tables", lambda n: fox.page_tables(i(2), n, i(2, 3), i(5), i(1), 16, 4), (i(2),)),
            ("release_pages", lambda n: fox.release_pages(i(2), n, i(2, 3), i(5), i(1), 16), (i(2),)),
            ("paged_update", lambda *a: fox.paged_update(*a, i(4)), (k, v, g, rows, rows.clone(), gates)),
            ("paged_forgetting_attention", lambda *a: fox.paged_forgetting_attention(*a, i(3, 4), i(3)), (q, k, v, g))]


@pytest.mark.parametrize("which", range(4))
def test_paged_operators_are_not_traced(which):
    """A trace would keep the first call's results for every input, and none of the writes."""
    name, f, args = paged_calls()[which]
    with torch.no_grad(), pytest.raises(_lib.FoxError, match=name + " cannot be traced"):
        torch.jit.trace(f, args, check_trace=False)


@pytest.mark.parametrize("which,at", [(2, i) for i in range(6)] + [(3, i) for i in range(4)])
def test_paged_operators_have_no_forward_mode(which, at):
    """A dual tensor, of values or of pages, raises: nothing comes back, or is written, without its tangent."""
    name, f, args = paged_calls()[which]
    with fwAD.dual_level(), torch.no_grad():
        args = [fwAD.make_dual(t, torch.ones_like(t)) if i == at else t for i, t in enumerate(args)]
        with pytest.raises(_lib.FoxError, match=name + " has no forward-mode"):
            f(*args)


def test_frequencies_have_no_forward_mode():
    with fwAD.dual_level(), torch.no_grad():
        f = fwAD.make_dual(F32, torch.ones_like(F32))
        with pytest.raises(_lib.FoxError, match="no forward-mode derivative for inv_freq"):
            fox.rotary_embedding(bf(1, 4, 2, 64), f)
        with pytest.raises(_lib.FoxError, match="no forward-mode derivative for inv_freq"):
            fox.qk_norm_rotary(bf(1, 4, 2, 64), bf(1, 4, 2, 64), torch.ones(64), torch.ones(64), f)


class Wrapper(torch.Tensor):
    """A subclass that holds no memory: its data pointer is the offset it was given."""

    @staticmethod
    def __new__(cls, t):
        return torch.Tensor._make_wrapper_subclass(cls, t.shape, strides=t.stride(), storage_offset=64, dtype=t.dtype, device=t.device)

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        raise RuntimeError(f"{func} was not meant to run")


@pytest.mark.parametrize("which,at", [(0, 0), (1, 0)] + [(2, i) for i in range(6)] + [(3, i) for i in range(4)])
def test_wrapped_tensors_never_reach_a_paged_kernel(which, at):
    _, f, args = paged_calls()[which]
    assert Wrapper(args[at]).data_ptr() == 64 * args[at].element_size()
    with torch.no_grad(), pytest.raises(_lib.FoxError, match="holds no memory"):
        f(*(Wrapper(t) if i == at else t for i, t in enumerate(args)))


@pytest.mark.parametrize("at", range(6))
def test_wrapped_tensors_never_reach_a_rotary_kernel(at):
    """Nor through the autograd functions, which take what the native nodes leave to them."""
    w = torch.ones(64)
    args = [bf(1, 4, 2, 64), bf(1, 4, 2, 64), w, w.clone(), F32, torch.zeros(4, dtype=torch.int32)]
    args[at] = Wrapper(args[at])
    calls = [lambda: fox.qk_norm_rotary(*args)]
    if at in (0, 4, 5):
        calls.append(lambda: fox.rotary_embedding(args[0], args[4], args[5]))
    for call in calls:
        with pytest.raises(_lib.FoxError, match="holds no memory"):
            call()


def test_frequencies_have_no_gradient_where_the_call_is_traced():
    f, w = F32.clone().requires_grad_(), torch.ones(64)
    with pytest.raises(_lib.FoxError, match="rotary_embedding has no gradient for inv_freq"):
        torch.jit.trace(lambda x: fox.rotary_embedding(x, f), (bf(1, 4, 2, 64),), check_trace=False)
    with pytest.raises(_lib.FoxError, match="qk_norm_rotary has no gradient for inv_freq"):
        torch.jit.trace(lambda x: fox.qk_norm_rotary(x, x, w, w, f), (bf(1, 4, 2, 64),), check_trace=False)


def test_history_ends_with_the_request():
    """What is asked for behind a request's end, in its last page or in pages that it does not own, is zero: not the rows of
    another request, nor what the memory held before."""
    c = fox.PagedFgateCache(num_layers=2, num_pages=4, page_size=16, num_heads=4, num_kv_heads=2, head_dim=16, max_requests=3,
                            max_length=64, device="cpu")
    for n, t in enumerate((c.k_pages, c.v_pages, c.gate_pages)):
        t.copy_((torch.arange(t.numel()).view(t.shape) % 997 + 1 + n).to(t.dtype))
    c.block_table[0, :2] = torch.tensor([2, 0], dtype=torch.int32)
    c.block_table[1, :1] = 3
    c.lengths.copy_(torch.tensor([21, 16, 0]))
    for request, ids, have in ((0, [2, 0], 21), (1, [3], 16), (2, [], 0)):
        for length in (0, have // 2, have, have + 1, 48, 64):
            got = c.history(1, request, length)
            n = min(have, length)
            for t, pool in zip(got, (c.k_pages, c.v_pages, c.gate_pages)):
                want = torch.cat([pool[1, p] for p in ids], 1)[:, :n] if ids else pool[1, 0, :, :0]
                assert t.shape == (1, pool.shape[2], length, *pool.shape[4:])
                assert torch.equal(t[0, :, :n], want) and not t[0, :, n:].any()
    c.block_table[0, 1] = 2 ** 30       # (an entry outside the pool: its keys take no part in the attention either)
    assert not c.history(0, 0, 21)[0][0, :, 16:].any()
    for length in (-1, 65):
        with pytest.raises(ValueError, match="0 to 64 tokens"):
            c.history(0, 0, length)


def test_module_refuses_its_first_call_in_a_capture(monkeypatch):
    """The copy from the host would end the capture; the refusal comes before it, and a device that has its copy needs none."""
    m, gpu = fox.RotaryEmbedding(64), torch.device("cuda", 0)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(_lib.FoxError, match="once before"):
        m.inv_freq(gpu)
    m._on_device[gpu] = F32
    assert m.inv_freq(gpu) is F32 and m.inv_freq(torch.device("cpu")).shape == (32,)


def test_ranges_of_a_launch():
    """The ranges that a backward's shares are counted by are those that its tokens are cut into."""
    lib = _lib.load()
    for B, T, H, Hk, D in ((3, 6001, 16, 16, 128), (3, 8003, 12, 4, 64), (1, 1, 1, 1, 16), (3, 10007, 24, 24, 16), (2, 8192, 33, 11, 128)):
        for half, interleaved in ((D // 2, 0), (D // 2, 1), (5, 0)):
            per = lib.fox_rotary_range(2, B, T, H + Hk, D, half, interleaved)
            assert lib.fox_qk_norm_rotary_partials(B, T, H, Hk, D) == -(-B * T // per)
    assert lib.fox_rotary_range(3, 1, 1, 1, 64, 32, 0) == 1 and lib.fox_rotary_range(0, 0, 1, 1, 64, 32, 0) == 1
    assert lib.fox_rotary_range(0, 2 ** 40, 2 ** 40, 1, 64, 32, 0) == 1 and lib.fox_rotary_range(0, 1, 1, 2 ** 40, 64, 32, 0) == 1


def test_expanded_gate_pages_are_not_written():
    """Several heads' gates in one place would leave any one of them there.  Reading such pages is allowed."""
    i = lambda *s: torch.zeros(*s, dtype=torch.int32)
    k, v, g = pages()
    for shared in (g[:, :1].expand(-1, 2, -1), g[:1].expand(5, -1, -1)):
        with pytest.raises(AssertionError, match="must not be expanded"):
            fox.paged_update(k, v, shared, bf(4, 2, 64), bf(4, 2, 64), torch.zeros(4, 2), i(4))
        with pytest.raises(_lib.FoxError, match="no CPU path"):
            fox.paged_forgetting_attention(bf(3, 2, 64), k, v, shared, i(3, 4), i(3))
