"""The 8-bit block operators on the CPU: definitions, refusals, modules."""
import copy

import pytest
import torch

from maggy_amd import ops
from maggy_amd.exceptions import HipExtensionMissingError  # noqa: F401
from maggy_amd.ops.block8 import groups8
from tests import _block8_oracle as oracle


def _normal(*shape, seed=0, std=1.0, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(*shape, generator=g).mul(std).to(dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16,
                                   torch.float32])
@pytest.mark.parametrize("R,C", [(1, 1), (3, 127), (5, 129), (2, 700),
                                 (300, 64)])
def test_pack_is_the_definition(R, C, dtype):
    x = _normal(R, C, dtype=dtype) * \
        torch.exp2(_normal(R, 1, seed=1) * 4).to(dtype)
    got = ops.unpack8(ops.pack8(x))
    assert torch.equal(got.double(), oracle.held(x).to(dtype).double())


def test_pack_extremes():
    x = torch.zeros(4, 200)
    x[0, 1], x[0, 2] = torch.finfo().max, 1.0
    x[1, 3], x[1, 4] = float("inf"), 2.0
    x[2, 5], x[2, 6] = float("nan"), -3.0
    got = ops.unpack8(ops.pack8(x))
    assert got[0, 1] == torch.finfo().max and got[0, 2] == 0
    assert got[1, 3].isnan() and got[1, 4] == 2
    assert got[2, 5].isnan() and got[2, 6] == -3
    assert torch.equal(got[3], x[3])


def test_held_bytes():
    h = ops.pack8(_normal(256, 512, dtype=torch.bfloat16))
    assert h.nbytes() == 256 * 512 + 256 * 4
    assert "Block8" in repr(h)


def test_swiglu8():
    g, u = (_normal(9, 300, seed=s).requires_grad_(True) for s in (1, 2))
    dh = _normal(9, 300, seed=3)
    h = ops.swiglu8(g, u)
    h.backward(dh)
    for got, (want, bound) in zip((h, g.grad, u.grad),
                                  oracle.swiglu(g.detach(), u.detach(), dh)):
        oracle.assert_within(got, want, bound)


def test_rms_norm8():
    x = _normal(9, 300, seed=1).requires_grad_(True)
    w = _normal(300, seed=2).requires_grad_(True)
    dy = _normal(9, 300, seed=3)
    y = ops.rms_norm8(x, w)
    y.backward(dy)
    for got, (want, bound) in zip(
            (y, x.grad, w.grad),
            oracle.rms(x.detach(), w.detach(), dy, 1e-5)):
        oracle.assert_within(got, want, bound)


@pytest.mark.parametrize("M,K,Ns", [(1, 64, (32,)), (17, 130, (77, 129)),
                                    (5, 300, (64, 1, 200, 3))])
def test_linear8(M, K, Ns):
    x = _normal(M, K, seed=1).requires_grad_(True)
    ws = [_normal(n, K, seed=2 + i, std=0.1).requires_grad_(True)
          for i, n in enumerate(Ns)]
    dys = [_normal(M, n, seed=8 + i) for i, n in enumerate(Ns)]
    ys = ops.linear8(x, *ws)
    ys = ys if isinstance(ys, tuple) else (ys,)
    grads = torch.autograd.grad(ys, [x, *ws], dys)
    want_y, want_dx, want_dw = oracle.linear(
        x.detach(), [w.detach() for w in ws], dys)
    for got, (want, bound) in zip(
            (*ys, *grads), (*want_y, want_dx, *want_dw)):
        oracle.assert_within(got, want, bound)
    with torch.no_grad():
        again = ops.linear8(x, ops.pack_weight8(*ws))
        again = again if isinstance(again, tuple) else (again,)
        for a, b in zip(again, ys):
            torch.testing.assert_close(a, b, rtol=1e-5, atol=1e-6)


def test_a_gradient_against_differences():
    """Where everything is exact in 8 bits the gradient is the slope."""
    # small whole numbers times a power of two fit e4m3 under any scale
    x = torch.randint(-7, 8, (6, 40), generator=torch.Generator()
                      .manual_seed(0)).float().requires_grad_(True)
    w = torch.randint(-7, 8, (5, 40), generator=torch.Generator()
                      .manual_seed(1)).float().requires_grad_(True)
    d = torch.randint(-7, 8, (6, 5), generator=torch.Generator()
                      .manual_seed(2)).float()
    ops.linear8(x, w).backward(d)

    def loss(x, w):
        return (ops.linear8(x, w) * d).sum()

    with torch.no_grad():
        for t, grad, other in ((x, x.grad, lambda t: loss(t, w)),
                               (w, w.grad, lambda t: loss(x, t))):
            for i, j in ((0, 0), (3, 17), (4, 39)):
                hi, lo = t.detach().clone(), t.detach().clone()
                hi[i, j] += 1
                lo[i, j] -= 1
                slope = (other(hi) - other(lo)) / 2
                assert slope == grad[i, j]


# ------------------------------------------------------------------ refusals
def test_refusals():
    x, w = _normal(4, 32), _normal(8, 32)
    with pytest.raises(TypeError):
        ops.pack8(x.double())
    with pytest.raises(TypeError):
        ops.pack8([1.0])
    with pytest.raises(ValueError):
        ops.pack8(torch.tensor(1.0))
    with pytest.raises(ValueError):
        ops.pack8(torch.zeros(3, 0))
    with pytest.raises(TypeError):
        ops.unpack8(x)
    with pytest.raises(TypeError):
        ops.unpack8(ops.pack8(x), torch.int32)
    with pytest.raises(ValueError):
        ops.swiglu8(x, x[:2])
    with pytest.raises(ValueError):
        ops.swiglu8(x, x.bfloat16())
    with pytest.raises(ValueError):
        ops.rms_norm8(x, torch.ones(31))
    with pytest.raises(ValueError):
        ops.linear8(x)
    with pytest.raises(ValueError):
        ops.linear8(x, *[w] * 5)
    with pytest.raises(ValueError):
        ops.linear8(x, _normal(8, 31))
    with pytest.raises(ValueError):
        ops.linear8(x, w, w[:, :16])
    with pytest.raises(ValueError):
        ops.linear8(x, w[:0])
    with pytest.raises(ValueError):
        ops.linear8(x, w[0])
    with pytest.raises(TypeError):
        ops.linear8(x, w.half())
    with pytest.raises(TypeError):
        ops.linear8(x, w.int())


def test_packed_weights_refuse_gradients_and_company():
    x, w = _normal(4, 32).requires_grad_(True), _normal(8, 32)
    packed = ops.pack_weight8(w)
    with pytest.raises(RuntimeError):
        ops.linear8(x, packed)
    with pytest.raises(TypeError):
        ops.linear8(x, packed, w)
    with pytest.raises(ValueError):
        ops.linear8(_normal(4, 31), packed)
    assert ops.linear8(x.detach(), packed).shape == (4, 8)


def test_second_derivatives_are_refused():
    x = _normal(4, 32).requires_grad_(True)
    w = _normal(8, 32).requires_grad_(True)
    y = ops.linear8(x, w)
    g, = torch.autograd.grad(y.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


# ------------------------------------------------------------------- modules
def test_modules_share_state_with_the_16_bit_ones():
    from maggy_amd.ops.linear import MaggyFeedForward

    torch.manual_seed(0)
    a, b = MaggyFeedForward(64, 96), ops.MaggyFeedForward8(64, 96)
    b.load_state_dict(a.state_dict())
    x = _normal(7, 64).requires_grad_(True)
    y = b(x)
    # 8 bits: 1/16 a value, far less over sums of 64
    assert (y - a(x)).norm() < 0.1 * a(x).norm()
    y.sum().backward()
    assert x.grad is not None
    assert all(p.grad is not None for p in b.parameters())
    c = copy.deepcopy(b)
    assert c.up8.linears[0] is c.w1 and c.up8.linears[0] is not b.w1


def test_module_packs_and_drops():
    lin = ops.MaggyLinear8(40, 30)
    x = _normal(3, 40)
    with torch.no_grad():
        before = lin(x)
        ops.pack8_model(lin)
        assert torch.equal(lin(x), before)
        assert lin.group.packed is not None
        ops.drop8_model(lin)
        assert lin.group.packed is None
        ops.pack8_model(lin)
        lin.weight.mul_(2)  # a changed weight is noticed
        assert torch.equal(lin(x), before * 2)
        assert lin.group.packed is None
        ops.pack8_model(lin)
        lin.weight = torch.nn.Parameter(lin.weight.detach() / 2)
        assert torch.equal(lin(x), before)
        ops.pack8_model(lin)
    lin(x)  # with gradients: the weights are about to change
    assert lin.group.packed is None
    with pytest.raises(ValueError):
        from maggy_amd.ops.block8 import Linear8Group

        Linear8Group(torch.nn.Linear(3, 3))


def test_norm_module():
    n = ops.MaggyRMSNorm8(48)
    x = _normal(5, 48).requires_grad_(True)
    n(x).sum().backward()
    assert n.weight.grad.shape == (48,) and x.grad.shape == x.shape


# --------------------------------------------------------------------- Llama
def _llama(eight_bit, seed=0):
    from maggy_amd.models import LlamaConfig, LlamaModel

    torch.manual_seed(seed)
    cfg = LlamaConfig.tiny(vocab_size=97)
    cfg.eight_bit = eight_bit
    return LlamaModel(cfg)


def test_llama_in_8_bits_is_near_the_16_bit_one():
    a, b = _llama(False), _llama(True)
    assert a.state_dict().keys() == b.state_dict().keys()
    b.load_state_dict(a.state_dict())
    tokens = torch.randint(0, 97, (2, 16))
    with torch.no_grad():
        want, got = a(tokens), b(tokens)
    assert (got - want).norm() < 0.1 * want.norm()
    la, lb = a(tokens, tokens), b(tokens, tokens)
    la.backward()
    lb.backward()
    for (name, p), q in zip(a.named_parameters(), b.parameters()):
        # 4 significant bits an operand: the gradients point the same way
        cos = torch.nn.functional.cosine_similarity(
            p.grad.flatten(), q.grad.flatten(), dim=0)
        assert cos > 0.95, (name, cos)


def test_llama_in_8_bits_decodes():
    from maggy_amd.ops.block8 import groups8

    m = _llama(True).eval()
    prompt = torch.randint(0, 97, (2, 5))
    out = m.generate(prompt, max_new_tokens=6)
    assert all(g.packed is None for g in groups8(m))  # dropped again
    assert len(groups8(m)) == 8
    seq = prompt
    with torch.no_grad():
        for _ in range(6):
            nxt = m(seq)[:, -1, :].argmax(-1, keepdim=True)
            seq = torch.cat([seq, nxt], 1)
    assert torch.equal(out, seq)
    ops.pack8_model(m)
    assert torch.equal(m.generate(prompt, max_new_tokens=6), out)
    assert all(g.packed is not None for g in groups8(m))  # the caller's
    got = m.generate_captured(prompt, max_new_tokens=6, use_graph=False)
    assert torch.equal(got, out)


@pytest.mark.parametrize("eight_bit", [False, True])
def test_masked_decoding_reads_no_memory_as_it_was(eight_bit, monkeypatch):
    m = _llama(eight_bit).eval()
    prompt = torch.randint(0, 97, (2, 5))
    want = m.generate(prompt, max_new_tokens=6)
    monkeypatch.setattr(
        torch.Tensor, "new_empty",
        lambda self, *size: self.new_full(size, float("nan")))
    got = m.generate_captured(prompt, max_new_tokens=6, use_graph=False)
    assert torch.equal(got, want)


def _group(N=48, K=96, dtype=torch.float32):
    torch.manual_seed(0)
    m = ops.MaggyLinear8(K, N).to(dtype)
    return m, torch.randn(3, K, dtype=dtype)


@torch.no_grad()
def test_packed_weights_of_a_converted_module_are_dropped():
    m, x = _group()
    ops.pack8_model(m)
    m.to(torch.bfloat16)
    y = m(x.bfloat16())
    assert m.group.packed is None
    assert torch.equal(y, ops.linear8(x.bfloat16(), m.weight))


@torch.no_grad()
def test_packed_module_copies():
    m, x = _group()
    ops.pack8_model(m)
    other = copy.deepcopy(m)
    other.weight.mul_(2)
    assert torch.equal(other(x), 2 * m(x))
    assert m.group.packed is not None


def test_weights_made_in_inference_mode_pack():
    with torch.inference_mode():
        m, x = _group()
        want = m(x)
        ops.pack8_model(m)
        assert torch.equal(m(x), want)
        assert m.group.packed is not None


@torch.no_grad()
def test_weights_changed_while_they_are_packed(monkeypatch):
    from maggy_amd.ops import block8

    m, x = _group()
    want = 2 * m(x)
    pack = block8.pack_weight8

    def changed_meanwhile(*weights):
        packed = pack(*weights)
        m.weight.mul_(2)
        return packed

    monkeypatch.setattr(block8, "pack_weight8", changed_meanwhile)
    ops.pack8_model(m)
    assert torch.equal(m(x), want)


@torch.no_grad()
def test_weights_dropped_by_another_thread_meanwhile(monkeypatch):
    m, x = _group()
    want = m(x)
    ops.pack8_model(m)
    state = m.group._state

    def dropped_meanwhile():
        m.group.drop()
        return state()

    monkeypatch.setattr(m.group, "_state", dropped_meanwhile)
    assert torch.equal(m(x), want)


def test_bench_refuses_8_bits_of_other_models(monkeypatch):
    bench = pytest.importorskip("bench")
    monkeypatch.setattr("sys.argv", ["bench.py", "--eight-bit"])
    with pytest.raises(SystemExit):
        bench.parse_args()
    monkeypatch.setattr("sys.argv", ["bench.py", "--eight-bit", "--model",
                                     "llama8b"])
    assert bench.parse_args().eight_bit


# ------------------------------------------ what a group's owner holds now
class _Doubled(torch.nn.Module):
    def __init__(self, linear):
        super().__init__()
        self.linear = linear

    def forward(self, x):
        return 2 * self.linear(x)


def _set(model, path, child):
    parent = model.get_submodule(path.rpartition(".")[0])
    setattr(parent, path.rpartition(".")[2], child)


@pytest.mark.parametrize("path", ["layers.0.attn.wq", "layers.0.attn.wo"])
@torch.no_grad()
def test_an_ablated_projection_is_gone(path):
    from maggy_amd.ablation.ablationstudy import drop_layers

    m = _llama(True).eval()
    tokens = torch.randint(0, 97, (2, 9))
    before = m(tokens)
    other = copy.deepcopy(m)
    attn = other.layers[0].attn
    if path.endswith("wq"):
        attn.qkv8 = lambda x: (x, *ops.linear8(x, attn.wk.weight,
                                               attn.wv.weight))
    else:
        attn.out8 = lambda x: x
    want = other(tokens)
    drop_layers(m, path)
    assert torch.equal(m(tokens), want) and not torch.equal(want, before)
    ops.pack8_model(m)
    assert torch.equal(m(tokens), want)
    assert torch.equal(m.generate(tokens, 3), m.generate_captured(
        tokens, 3, use_graph=False))


@pytest.mark.parametrize("path", ["layers.0.attn.wk", "layers.1.attn.wo",
                                  "layers.0.ffn.w1", "layers.0.ffn.w3",
                                  "layers.1.ffn.w2"])
def test_a_replaced_linear_is_the_one_that_runs(path):
    m = _llama(True)
    other = copy.deepcopy(m)
    tokens = torch.randint(0, 97, (2, 9))
    old = m.get_submodule(path)
    new = torch.nn.Linear(old.in_features, old.out_features, bias=False)
    _set(m, path, new)
    with torch.no_grad():
        other.get_submodule(path).weight.copy_(new.weight)
        want = other(tokens)
        assert torch.equal(m(tokens), want)
        ops.pack8_model(m)
        assert torch.equal(m(tokens), want)
    m(tokens).sum().backward()
    assert new.weight.grad is not None and old.weight.grad is None
    # every parameter that is listed takes part
    assert all(p.grad is not None for p in m.parameters())


def test_an_adapter_around_a_linear_runs():
    m = _llama(True)
    other = copy.deepcopy(m)
    tokens = torch.randint(0, 97, (2, 9))
    attn, theirs = m.layers[0].attn, other.layers[0].attn
    v = torch.nn.Linear(*attn.wv.weight.t().shape, bias=False)
    o = torch.nn.Linear(*attn.wo.weight.t().shape, bias=False)
    attn.wv, attn.wo = _Doubled(v), _Doubled(o)
    theirs.qkv8 = lambda x: (*ops.linear8(x, theirs.wq.weight,
                                          theirs.wk.weight), 2 * v(x))
    theirs.out8 = lambda x: 2 * o(x)
    assert torch.equal(m(tokens), other(tokens))
    m(tokens).sum().backward()
    assert all(p.grad is not None for p in m.parameters())


@torch.no_grad()
def test_a_linear_with_a_bias_and_one_of_another_type_run():
    ff = ops.MaggyFeedForward8(64, 96)
    x = _normal(5, 64)
    biased = torch.nn.Linear(96, 64)
    ff.w2 = biased
    want = biased(ops.swiglu8(*ops.linear8(x, ff.w1.weight, ff.w3.weight)))
    assert torch.equal(ff(x), want)
    ff.w3.bfloat16()  # not of w1's type: not one product with it
    want = biased(ops.swiglu8(ops.linear8(x, ff.w1.weight),
                              ops.linear8(x, ff.w3.weight)))
    assert torch.equal(ff(x), want)
    ops.pack8_model(ff)
    assert torch.equal(ff(x), want)
    lin = ops.MaggyLinear8(40, 30)
    lin.bias = torch.nn.Parameter(torch.ones(30))
    with pytest.raises(ValueError, match="bias"):
        lin(_normal(3, 40))


@torch.no_grad()
def test_a_module_that_extends_the_8_bit_linear():
    class Doubled(ops.MaggyLinear8):
        def forward(self, x):
            return 2 * super().forward(x)

    m, x = Doubled(40, 30), _normal(3, 40)
    want = 2 * ops.linear8(x, m.weight)
    assert torch.equal(m(x), want)
    ops.pack8_model(m)
    assert torch.equal(m(x), want) and m.group.packed is not None


@pytest.mark.parametrize("path", ["layers.0.attn.wq", "layers.0.attn.wo",
                                  "layers.1.ffn.w1", "layers.1.ffn.w2"])
@torch.no_grad()
def test_hooks_of_a_linear_run(path):
    m = _llama(True).eval()
    tokens = torch.randint(0, 97, (2, 9))
    want, seen = m(tokens), []
    lin = m.get_submodule(path)
    for packed in (False, True):
        if packed:
            ops.pack8_model(m)
        hooks = [lin.register_forward_pre_hook(
                     lambda mod, args: seen.append(args[0])),
                 lin.register_forward_hook(
                     lambda mod, args, out: seen.append(out))]
        assert torch.equal(m(tokens), want)  # seen, and still in 8 bits
        x, y = seen
        assert torch.equal(y, ops.linear8(x, lin.weight))
        for h in hooks:
            h.remove()
        seen.clear()
        hook = lin.register_forward_hook(lambda mod, args, out: 0 * out)
        assert not torch.equal(m(tokens), want)
        hook.remove()
        assert torch.equal(m(tokens), want) and not seen
    # the group read its packed weights again
    assert all(g.packed is not None for g in groups8(m))


def test_hooks_of_all_modules_and_of_gradients_run():
    from torch.nn.modules import module as every

    ff, seen = ops.MaggyFeedForward8(64, 96), []
    x = _normal(5, 64).requires_grad_(True)
    hook = every.register_module_forward_hook(
        lambda mod, args, out: seen.append(mod))
    ff(x)
    hook.remove()
    assert all(any(m is s for s in seen) for m in (ff.w1, ff.w2, ff.w3))
    hook = ff.w3.register_full_backward_hook(
        lambda mod, dx, dy: seen.append(dy[0]))
    seen.clear()
    ff(x).sum().backward()
    assert len(seen) == 1 and seen[0].shape == (5, 96)
    hook.remove()


def test_a_pruned_linear_trains():
    from torch.nn.utils import prune

    ff, x = ops.MaggyFeedForward8(64, 96), _normal(5, 64)
    prune.l1_unstructured(ff.w1, "weight", amount=0.5)
    mask = ff.w1.weight_mask
    for _ in range(3):
        y = ff(x)
        y.sum().backward()
        grad = ff.w1.weight_orig.grad
        assert grad is not None and (grad[mask == 0] == 0).all()
        with torch.no_grad():
            for p in ff.parameters():
                p -= 0.1 * p.grad
                p.grad = None
    with torch.no_grad():
        want = ops.linear8(ops.swiglu8(*ops.linear8(
            x, ff.w1.weight_orig * mask, ff.w3.weight)), ff.w2.weight)
        assert torch.equal(ff(x), want)


@torch.no_grad()
def test_a_parametrized_and_a_patched_linear_run():
    from torch.nn.utils import parametrize

    class Halved(torch.nn.Module):
        def forward(self, w):
            return w / 2

    ff, x = ops.MaggyFeedForward8(64, 96), _normal(5, 64)
    parametrize.register_parametrization(ff.w3, "weight", Halved())
    ff.w2.forward = lambda x: x
    for _ in range(2):
        g, u = ops.linear8(x, ff.w1.weight, ff.w3.weight)
        want = ops.swiglu8(g, u)
        assert torch.equal(ff(x), want)
        ops.pack8_model(ff)
        ff.w3.parametrizations.weight.original.mul_(3)


# ------------------------------------------------- packing while it decodes
@pytest.fixture
def packings(monkeypatch):
    """How many weights were put in 8 bits, by a pack or on the way."""
    from maggy_amd.ops import block8

    count, held = [], block8._held_weight

    def counted(w):
        count.append(w.shape)
        return held(w)

    monkeypatch.setattr(block8, "_held_weight", counted)
    return count


def _decode(m, prompt, captured):
    if captured:
        return m.generate_captured(prompt, 9, use_graph=False)
    return m.generate(prompt, 9)


@pytest.mark.parametrize("captured", [False, True])
def test_changed_weights_are_packed_once_a_decode(captured, packings):
    m = _llama(True).eval()
    prompt = torch.randint(0, 97, (2, 5))
    _decode(m, prompt, captured)
    once = len(packings)
    assert once == 14  # seven a layer
    ops.pack8_model(m)
    with torch.no_grad():
        for p in m.parameters():
            p.mul_(1.5)
    packings.clear()
    got = _decode(m, prompt, captured)
    assert len(packings) == once
    ops.drop8_model(m)
    assert torch.equal(got, _decode(m, prompt, captured))


@pytest.mark.parametrize("captured", [False, True])
def test_decodes_of_two_threads_pack_once_each(captured, packings):
    import threading

    m = _llama(True).eval()
    prompt = torch.randint(0, 97, (2, 5))
    want = _decode(m, prompt, captured)
    once, inside, done = len(packings), threading.Event(), threading.Event()
    packings.clear()

    class Waits(torch.nn.Module):
        def forward(self, x):
            if threading.current_thread() is other:
                inside.set()
                assert done.wait(60)
            return x

    # the other thread stops in the middle of its decode
    m.norm = torch.nn.Sequential(Waits(), m.norm)
    got = []
    other = threading.Thread(
        target=lambda: got.append(_decode(m, prompt, captured)))
    other.start()
    try:
        assert inside.wait(60)
        mine = _decode(m, prompt, captured)
        assert len(packings) == 2 * once
    finally:
        done.set()
        other.join()
    assert torch.equal(mine, want) and torch.equal(got[0], want)
    assert len(packings) == 2 * once
    assert all(g.packed is None for g in groups8(m))


def test_a_decode_leaves_what_others_packed_meanwhile():
    m = _llama(True).eval()
    prompt = torch.randint(0, 97, (2, 5))
    norm = m.norm

    class Packs(torch.nn.Module):
        def forward(self, x):
            ops.pack8_model(m)
            m.norm = norm
            return norm(x)

    m.norm = Packs()
    got = m.generate(prompt, 6)
    assert all(g.packed is not None for g in groups8(m))
    assert torch.equal(m.generate(prompt, 6), got)


# ---------------------------------------- weights written by the framework
def _zero_rank(rank, path):
    import torch.distributed as dist

    from maggy_amd.parallel.zero import ZeroFusedSGD, broadcast_module_params

    dist.init_process_group("gloo", init_method="file://" + path, rank=rank,
                            world_size=2)
    torch.manual_seed(rank)
    m = torch.nn.Sequential(*[ops.MaggyLinear8(32, 32) for _ in range(3)])
    x = _normal(4, 32)

    def agrees():
        with torch.no_grad():
            want = x
            for lin in m:
                want = ops.linear8(want, lin.weight)
            assert torch.equal(m(x), want)

    ops.pack8_model(m)
    broadcast_module_params(m)
    agrees()
    opt = ZeroFusedSGD(list(m.parameters()), lr=0.5)
    m(x).square().sum().backward()
    ops.pack8_model(m)  # between the gradients and the step
    opt.step()
    agrees()
    dist.destroy_process_group()


@pytest.mark.timeout(120)
def test_packed_weights_that_another_rank_updates(tmp_path):
    torch.multiprocessing.spawn(_zero_rank, (str(tmp_path / "store"),), 2)


@torch.no_grad()
def test_weights_written_behind_torch_while_they_are_packed(monkeypatch):
    from maggy_amd.ops import block8

    m, x = _group()
    want = 2 * m(x)
    pack = block8.pack_weight8

    def written_meanwhile(*weights):
        packed = pack(*weights)
        m.weight.data.mul_(2)
        block8.weights_written(m.parameters())
        return packed

    monkeypatch.setattr(block8, "pack_weight8", written_meanwhile)
    ops.pack8_model(m)
    assert torch.equal(m(x), want)


# ------------------------------------------------- forward-mode derivatives
def _forward_mode_calls(x, w, n):
    packed = ops.pack_weight8(w)
    return [lambda t: ops.swiglu8(t, x), lambda t: ops.swiglu8(x, t),
            lambda t: ops.rms_norm8(t, n), lambda t: ops.linear8(t, w),
            lambda t: ops.linear8(t, w, w), lambda t: ops.linear8(t, packed)]


@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_is_refused(grad):
    from torch.autograd import forward_ad

    x, w, n = _normal(4, 32), _normal(8, 32), torch.ones(32)
    with torch.set_grad_enabled(grad), forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        for call in _forward_mode_calls(x, w, n):
            with pytest.raises((RuntimeError, NotImplementedError)):
                call(dual)
            call(x)
        with pytest.raises((RuntimeError, NotImplementedError)):
            ops.linear8(x, forward_ad.make_dual(w, torch.ones_like(w)))
        with pytest.raises((RuntimeError, NotImplementedError)):
            ops.rms_norm8(x, forward_ad.make_dual(n, torch.ones_like(n)))


# ------------------------------------------------------------------ launches
def _launchers():
    """The extension's launch functions, and a call of each on rows of one
    value and no memory."""
    import ctypes

    if not ops.has_ext():
        pytest.skip("the extension is not built")
    lib = ctypes.CDLL(ops.require_ext().__file__)
    i, n, p = ctypes.c_int, ctypes.c_longlong, ctypes.c_void_p
    # r stands for the number of rows
    r = type("Rows", (n,), {})
    calls = {
        "launch_b8_pack": (i, i, p, n, r, i, p, i, p, n, p),
        "launch_b8_unpack": (i, i, p, i, p, n, r, i, p, p),
        "launch_b8_swiglu_fwd": (i, i, p, n, p, n, r, i, p, p, p, i, p, p, n,
                                 p),
        "launch_b8_swiglu_bwd": (i, i, p, n, p, p, i, p, p, n, r, i, p, p, p),
        "launch_b8_rms_fwd": (i, i, p, n, p, r, i, ctypes.c_float, p, p, p, i,
                              p, n, p),
        "launch_b8_rms_bwd": (i, i, p, n, p, i, p, n, p, p, r, i, p, p, p, p)}

    def call(name, rows):
        f, types = getattr(lib, name), calls[name]
        f.restype = i
        f.argtypes = [n if t is r else t for t in types]
        return f(*(None if t is p else rows if t is r else 1 for t in types))

    return lib, list(calls), call


@pytest.mark.skipif(torch.cuda.is_available(),
                    reason="without a GPU every launch is refused")
def test_a_refused_launch_is_reported():
    _, names, call = _launchers()
    for name in names:
        assert call(name, 1) != 0, name
