"""The 8-bit block operators' kernels against 64-bit definitions (GPU)."""
import pytest
import torch

from maggy_amd import ops
from tests import _block8_oracle as oracle

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip("needs an AMD GPU", allow_module_level=True)

TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(shape, seed, std=1.0, dtype=torch.bfloat16):
    t = torch.empty(shape, device="cuda", dtype=torch.float32)
    return t.normal_(0.0, std, generator=_gen(seed)).to(dtype)


def _loud(R, C, seed, dtype=torch.bfloat16):
    """Rows and columns of very different size, some values zero."""
    x = _normal((R, C), seed, dtype=torch.float32)
    x *= torch.exp2(torch.randint(-12, 8, (R, 1), device="cuda",
                                  generator=_gen(seed + 1)).float())
    x *= torch.exp(_normal((1, C), seed + 2, dtype=torch.float32))
    x[_normal((R, C), seed + 3, dtype=torch.float32) > 1.5] = 0
    return x.to(dtype)


# -------------------------------------------------------------- pack, unpack
SHAPES = [(1, 1), (1, 128), (3, 127), (5, 129), (2, 512), (7, 640), (33, 1000),
          (257, 2048), (64, 14336), (1, 16384)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("R,C", SHAPES)
def test_pack_is_the_definition(R, C, dtype):
    x = _loud(R, C, R * 7 + C, dtype)
    got = ops.unpack8(ops.pack8(x))
    want = oracle.held(x)
    assert got.dtype == dtype
    assert torch.equal(got.double(), want.to(dtype).double())


def test_pack_ties_and_every_code():
    # every finite e4m3 value, the midpoints and their neighbours
    codes = torch.arange(127, device="cuda", dtype=torch.uint8)
    v = codes.view(torch.float8_e4m3fn).double()
    mid = (v[1:] + v[:-1]) / 2
    x = torch.cat([v, mid, mid * (1 + 2 ** -20), mid * (1 - 2 ** -20)])
    x = torch.cat([x, -x]).float()
    x = torch.nn.functional.pad(x, (0, -len(x) % 127)).view(-1, 127)
    top = torch.full((x.shape[0], 1), 448.0, device="cuda")
    x = torch.cat([x, top], 1)  # scale 1 in every block
    for scale in (1.0, 2.0 ** -100, 2.0 ** 60):
        got = ops.unpack8(ops.pack8(x * scale))
        assert torch.equal(got.double(), oracle.held(x * scale))


@pytest.mark.parametrize("dtype", TYPES)
def test_pack_extremes(dtype):
    info = torch.finfo(dtype)
    x = torch.zeros(8, 300, device="cuda", dtype=dtype)
    x[1, 3] = info.max
    x[1, 4] = -info.max
    x[2] = info.smallest_normal
    x[3, ::2] = info.tiny / 4  # subnormal
    x[4, 5] = float("inf")
    x[4, 130] = float("-inf")
    x[4, 6] = 1.5
    x[5, 7] = float("nan")
    x[5, 8] = -2.5
    x[6] = float("nan")
    x[7] = 448.0
    got = ops.unpack8(ops.pack8(x)).double()
    want = oracle.held(x).clamp(-info.max, info.max).to(dtype).double()
    assert torch.equal(got.nan_to_num(7777), want.nan_to_num(7777))


@pytest.mark.parametrize("dtype", TYPES)
def test_pack_strides(dtype):
    x = _loud(40, 600, 5, dtype)
    for v in (x[:, 3:], x[::3, :256], x.t(), x[:, ::2], x[:1].expand(9, 600),
              x.view(4, 10, 600)[:, ::2], x[:0], x[:, 7:8]):
        flat = v.reshape(-1, v.shape[-1])
        got = ops.unpack8(ops.pack8(v))
        assert got.shape == v.shape
        assert torch.equal(got.reshape(flat.shape).double(),
                           oracle.held(flat).to(dtype).double())


def test_pack_cpu_and_gpu_hold_the_same_bytes():
    x = _loud(37, 1000, 11)
    a, b = ops.pack8(x), ops.pack8(x.cpu())
    assert torch.equal(a.codes.cpu(), b.codes)
    assert torch.equal(a.scales[:, :37].cpu(), b.scales[:, :37])


# -------------------------------------------------------------------- swiglu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("R,C", [(1, 1), (1, 4096), (3, 129), (37, 1000),
                                 (130, 512), (65, 14336)])
def test_swiglu8(R, C, dtype):
    g = _normal((R, C), 1, 2.0, dtype).requires_grad_(True)
    u = _normal((R, C), 2, 1.0, dtype).requires_grad_(True)
    dh = _normal((R, C), 3, 1.0, dtype)
    h = ops.swiglu8(g, u)
    h.backward(dh)
    for got, (want, bound) in zip((h, g.grad, u.grad),
                                  oracle.swiglu(g.detach(), u.detach(), dh)):
        oracle.assert_within(got, want, bound)
    with torch.no_grad():
        assert torch.equal(ops.swiglu8(g, u), h)


def test_swiglu8_far_values():
    v = torch.tensor([0.0, -0.0, 1e-30, -1e-30, 20, -20, 90, -90, 3e4, -3e4,
                      1e30, -1e30], device="cuda")
    for dtype in (torch.bfloat16, torch.float32):
        g = v.to(dtype)[:, None].repeat(1, 128).requires_grad_(True)
        u = torch.ones_like(g).requires_grad_(True)
        h = ops.swiglu8(g, u)
        h.backward(torch.ones_like(h))
        for got, (want, bound) in zip(
                (h, g.grad, u.grad),
                oracle.swiglu(g.detach(), u.detach(), torch.ones_like(g))):
            oracle.assert_within(got, want, bound + 1e-30)


def test_swiglu8_strided_halves():
    both = _normal((50, 2, 700), 4).requires_grad_(True)
    g, u = both[:, 0], both[:, 1]
    dh = _normal((50, 700), 5)
    ops.swiglu8(g, u).backward(dh)
    want = oracle.swiglu(g.detach(), u.detach(), dh)
    oracle.assert_within(both.grad[:, 0], *want[1])
    oracle.assert_within(both.grad[:, 1], *want[2])


# ----------------------------------------------------------------------- rms
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("R,C", [(1, 1), (7, 2050), (5, 64), (600, 129),
                                 (2100, 513), (33, 1024), (1030, 2048),
                                 (700, 4096), (9, 8191), (12, 16384)])
def test_rms_norm8(R, C, dtype):
    x = _normal((R, C), 1, 3.0, dtype).requires_grad_(True)
    w = (1 + 0.2 * _normal((C,), 2, dtype=torch.float32)).requires_grad_(True)
    dy = _normal((R, C), 3, 1.0, dtype)
    y = ops.rms_norm8(x, w, 1e-5)
    y.backward(dy)
    for got, (want, bound) in zip(
            (y, x.grad, w.grad),
            oracle.rms(x.detach(), w.detach(), dy, 1e-5)):
        oracle.assert_within(got, want, bound)
    with torch.no_grad():
        assert torch.equal(ops.rms_norm8(x, w, 1e-5), y)


def test_rms_norm8_partial_gradients_and_zero_rows():
    x = _normal((6, 300), 1)
    x[2] = 0
    w = torch.ones(300, device="cuda")
    dy = _normal((6, 300), 2)
    want = oracle.rms(x, w, dy, 1e-5)
    xg = x.clone().requires_grad_(True)
    ops.rms_norm8(xg, w).backward(dy)
    oracle.assert_within(xg.grad, *want[1])
    wg = w.clone().requires_grad_(True)
    ops.rms_norm8(x, wg).backward(dy)
    oracle.assert_within(wg.grad, *want[2])
    empty = x[:0].requires_grad_(True)
    out = ops.rms_norm8(empty, wg)
    wg.grad = None
    out.sum().backward()
    assert out.shape == (0, 300) and torch.equal(wg.grad,
                                                 torch.zeros_like(wg))


# -------------------------------------------------------------------- linear
LINEAR = [(1, 64, (32,)), (1, 2048, (2048,)), (8, 4096, (512,)),
          (17, 128, (16,)), (33, 130, (77, 129)), (128, 128, (128,)),
          (130, 515, (64, 64, 64, 1)), (256, 512, (256,)),
          (300, 1111, (777,)), (513, 640, (384, 130)), (1000, 256, (256,)),
          (1, 1, (1,))]


def _linear_inputs(M, K, Ns, wtype=torch.bfloat16, seed=0):
    x = _normal((M, K), seed)
    x = (x.float() * torch.exp(_normal((1, K), seed + 1,
                                       dtype=torch.float32))).bfloat16()
    ws = [_normal((n, K), seed + 2 + i, 0.05, wtype)
          for i, n in enumerate(Ns)]
    dys = [_normal((M, n), seed + 9 + i, 1e-3) for i, n in enumerate(Ns)]
    return x, ws, dys


def _check_linear(x, ws, dys):
    x = x.detach().requires_grad_(True)
    ws = [w.detach().requires_grad_(True) for w in ws]
    ys = ops.linear8(x, *ws)
    ys = ys if isinstance(ys, tuple) else (ys,)
    grads = torch.autograd.grad(ys, [x, *ws], dys)
    want_y, want_dx, want_dw = oracle.linear(
        x.detach(), [w.detach() for w in ws], dys)
    for i, (y, (want, bound)) in enumerate(zip(ys, want_y)):
        assert y.is_contiguous()
        oracle.assert_within(y, want, bound, "y{}".format(i))
    oracle.assert_within(grads[0], *want_dx, "dx")
    for i, (d, (want, bound)) in enumerate(zip(grads[1:], want_dw)):
        assert d.dtype == ws[i].dtype and d.is_contiguous()
        oracle.assert_within(d, want, bound, "dw{}".format(i))
    return ys


@pytest.mark.parametrize("M,K,Ns", LINEAR)
def test_linear8(M, K, Ns):
    x, ws, dys = _linear_inputs(M, K, Ns)
    ys = _check_linear(x, ws, dys)
    with torch.no_grad():
        packed = ops.pack_weight8(*ws)
        for call in (ops.linear8(x, packed), ops.linear8(x, *ws)):
            call = call if isinstance(call, tuple) else (call,)
            for a, b in zip(call, ys):
                assert torch.equal(a, b)


def test_linear8_fp32_weights():
    _check_linear(*_linear_inputs(200, 300, (140, 100), torch.float32))


def test_linear8_strides_and_leading_axes():
    x, ws, dys = _linear_inputs(60, 400, (150,))
    wide = torch.zeros(60, 500, device="cuda", dtype=torch.bfloat16)
    wide[:, 50:450] = x
    want, = _check_linear(x, ws, dys)
    with torch.no_grad():
        assert torch.equal(ops.linear8(wide[:, 50:450], ws[0]), want)
        assert torch.equal(ops.linear8(x.t().contiguous().t(), ws[0]), want)
        turned = ws[0].t().contiguous().t()
        assert torch.equal(ops.linear8(x, turned), want)
        out = ops.linear8(x.view(3, 20, 400), ws[0])
        assert out.shape == (3, 20, 150)
        assert torch.equal(out.view(60, 150), want)
        assert ops.linear8(x[:0], ws[0]).shape == (0, 150)


def test_linear8_bad_values_stay_in_their_rows():
    x, ws, _ = _linear_inputs(40, 300, (90,))
    with torch.no_grad():
        clean = ops.linear8(x, ws[0])
        x[7, 10] = float("inf")
        x[9, 299] = float("nan")
        got = ops.linear8(x, ws[0])
    bad = torch.zeros(40, dtype=torch.bool, device="cuda")
    bad[[7, 9]] = True
    assert got[bad].isnan().all()
    assert torch.equal(got[~bad], clean[~bad])


def test_linear8_only_the_gradients_asked_for():
    x, ws, dys = _linear_inputs(70, 200, (60, 50))
    want_y, want_dx, want_dw = oracle.linear(x, ws, dys)
    xg = x.clone().requires_grad_(True)
    torch.autograd.backward(ops.linear8(xg, *ws), dys)
    oracle.assert_within(xg.grad, *want_dx)
    second = ws[1].clone().requires_grad_(True)
    torch.autograd.backward(ops.linear8(x, ws[0], second), dys)
    oracle.assert_within(second.grad, *want_dw[1])
    # one output unused: its gradient is zero
    xg.grad = None
    ops.linear8(xg, *ws)[1].backward(dys[1])
    _, only, _ = oracle.linear(x, ws[1:], dys[1:])
    oracle.assert_within(xg.grad, *only)


def test_linear8_zero_rows_trains():
    x, ws, _ = _linear_inputs(1, 200, (60, 50))
    x = x[:0].requires_grad_(True)
    ws = [w.requires_grad_(True) for w in ws]
    a, b = ops.linear8(x, *ws)
    (a.sum() + b.sum()).backward()
    assert x.grad.shape == (0, 200)
    assert all(torch.equal(w.grad, torch.zeros_like(w)) for w in ws)


def test_results_repeat():
    x, ws, dys = _linear_inputs(600, 1000, (700,))
    runs = []
    for _ in range(2):
        xg = x.clone().requires_grad_(True)
        w = ws[0].clone().requires_grad_(True)
        n = torch.ones(1000, device="cuda", requires_grad=True)
        y = ops.linear8(ops.rms_norm8(xg, n), w)
        y.backward(dys[0])
        runs.append((y, xg.grad, w.grad, n.grad))
    for a, b in zip(*runs):
        assert torch.equal(a, b)


def test_another_stream():
    x, ws, dys = _linear_inputs(300, 500, (400,))
    want, = _check_linear(x, ws, dys)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s), torch.no_grad():
        got = ops.linear8(x, ws[0])
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want)


# -------------------------------------------------------- a run of them
def test_feed_forward_stage_by_stage():
    """Norm, gate and up, SwiGLU and down as a block runs them; every stage
    is checked on the inputs and gradients that it really had."""
    M, D, F = 200, 384, 640
    x = _normal((M, D), 1, 2.0).requires_grad_(True)
    nw = (1 + 0.1 * _normal((D,), 2, dtype=torch.float32)) \
        .requires_grad_(True)
    w1, w3 = (_normal((F, D), s, 0.05).requires_grad_(True) for s in (3, 4))
    w2 = _normal((D, F), 5, 0.05).requires_grad_(True)
    dy = _normal((M, D), 6, 1e-2)
    n = ops.rms_norm8(x, nw)
    g, u = ops.linear8(n, w1, w3)
    h = ops.swiglu8(g, u)
    y = ops.linear8(h, w2)
    inner = [n, g, u, h]
    for t in inner:
        t.retain_grad()
    y.backward(dy)
    d = [t.detach() for t in (x, nw, n, g, u, h, w1, w3, w2)]
    xd, nwd, nd, gd, ud, hd, w1d, w3d, w2d = d

    (want_y,), want_dh, (want_dw2,) = oracle.linear(hd, [w2d], [dy])
    oracle.assert_within(y, *want_y, "y")
    oracle.assert_within(h.grad, *want_dh, "dh")
    oracle.assert_within(w2.grad, *want_dw2, "dw2")
    for got, want in zip((h, g.grad, u.grad),
                         oracle.swiglu(gd, ud, h.grad)):
        oracle.assert_within(got, *want, "swiglu")
    ys, dn, dws = oracle.linear(nd, [w1d, w3d], [g.grad, u.grad])
    for got, want in zip((g, u, n.grad, w1.grad, w3.grad), (*ys, dn, *dws)):
        oracle.assert_within(got, *want, "gate and up")
    for got, want in zip((n, x.grad, nw.grad),
                         oracle.rms(xd, nwd, n.grad, 1e-5)):
        oracle.assert_within(got, *want, "norm")


def _llama(**kw):
    from maggy_amd.models import LlamaConfig, LlamaModel

    torch.manual_seed(0)
    cfg = LlamaConfig(vocab_size=256, dim=512, n_layers=2, n_heads=8,
                      n_kv_heads=4, ffn_hidden=704, max_seq_len=64,
                      eight_bit=True, **kw)
    with torch.device("cuda"):
        m = LlamaModel(cfg)
    m = m.to(torch.bfloat16)
    m.rope_cos, m.rope_sin = m.rope_cos.float(), m.rope_sin.float()
    return m


def test_llama_in_8_bits_trains_and_decodes():
    m = _llama()
    tokens = torch.randint(0, 256, (4, 33), device="cuda")
    loss = m(tokens[:, :-1], tokens[:, 1:].contiguous())
    loss.backward()
    for name, p in m.named_parameters():
        assert p.grad is not None and p.grad.isfinite().all(), name
        assert p.grad.abs().max() > 0, name
    out = m.generate(tokens[:, :8], max_new_tokens=6)
    ops.pack8_model(m)
    assert torch.equal(m.generate(tokens[:, :8], max_new_tokens=6), out)
    with torch.no_grad():
        packed = m(tokens)
        ops.drop8_model(m)
        assert torch.equal(m(tokens), packed)


def test_llama_in_8_bits_decodes_in_a_graph():
    """Like the 16-bit one in a process of its own, since captures depend on
    what else a process has run; the same step runs eagerly beside it."""
    import os
    import subprocess
    import sys

    code = (
        "import torch\n"
        "from tests.test_block8_gpu import _llama\n"
        "from maggy_amd import ops\n"
        "m = _llama().eval()\n"
        "prompt = torch.randint(0, 97, (2, 8), device='cuda')\n"
        "ref = m.generate_captured(prompt, 9, use_graph=False)\n"
        "assert torch.equal(m.generate_captured(prompt, 9), ref)\n"
        "ops.pack8_model(m)\n"
        "assert torch.equal(m.generate_captured(prompt, 9), ref)\n"
        "print('CAPTURED_OK')\n"
    )
    repo = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    p = subprocess.run([sys.executable, "-c", code], cwd=repo,
                       capture_output=True, text=True, timeout=100)
    assert p.returncode == 0 and "CAPTURED_OK" in p.stdout, \
        p.stdout[-1500:] + p.stderr[-1500:]


def test_under_autocast_from_fp32():
    lin = ops.MaggyLinear8(200, 100).cuda()
    x = _normal((50, 200), 1, dtype=torch.float32).requires_grad_(True)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y = lin(x)
    assert y.dtype == torch.bfloat16
    y.float().sum().backward()
    assert x.grad.dtype == torch.float32
    assert lin.weight.grad.dtype == torch.float32
    dys = [torch.ones_like(y)]
    want_y, want_dx, want_dw = oracle.linear(
        x.detach().bfloat16(), [lin.weight.detach()], dys)
    oracle.assert_within(y, *want_y[0])
    oracle.assert_within(x.grad.bfloat16(), *want_dx)
    oracle.assert_within(lin.weight.grad, *want_dw[0])


# -------------------------------------------------------------- graphs
def _replays(make, fill, seeds=(1, 2, 3, 4)):
    """Capture ``make()`` once, then replay it on the inputs of each seed
    between eager work, comparing every replay with the eager result."""
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        fill(0)
        make()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = make()
    for seed in seeds:
        fill(seed)
        graph.replay()
        got = [t.detach().clone() for t in outs]
        torch.cuda.synchronize()
        want = make()
        for a, b in zip(got, want):
            assert torch.equal(a, b), seed


def test_serving_in_a_graph():
    x = torch.zeros(4, 700, device="cuda", dtype=torch.bfloat16)
    with torch.no_grad():
        packed = ops.pack_weight8(_normal((300, 700), 1, 0.05),
                                  _normal((520, 700), 2, 0.05))

        def make():
            a, b = ops.linear8(x, packed)
            return a, b, ops.unpack8(ops.pack8(a))

        _replays(make, lambda seed: x.copy_(_normal((4, 700), seed)))


def test_training_in_a_graph():
    x = torch.zeros(150, 256, device="cuda",
                    dtype=torch.bfloat16).requires_grad_(True)
    nw = torch.ones(256, device="cuda", requires_grad=True)
    ws = [_normal((200, 256), s, 0.05).requires_grad_(True) for s in (3, 4)]
    dy = _normal((150, 200), 5)

    def make():
        g, u = ops.linear8(ops.rms_norm8(x, nw), *ws)
        h = ops.swiglu8(g, u)
        return (h.detach(),
                *torch.autograd.grad(h, [x, nw, *ws], dy))

    def fill(seed):
        with torch.no_grad():
            x.copy_(_normal((150, 256), seed))

    _replays(make, fill)


def test_two_graphs_do_not_share_workspaces():
    """Two captured calls, replayed in turn on two streams."""
    ins = [_normal((64, 2048), s) for s in (1, 2)]
    w = _normal((500, 2048), 3, 0.05)
    graphs, outs, want = [], [], []
    with torch.no_grad():
        packed = ops.pack_weight8(w)
        for x in ins:
            want.append(ops.linear8(x, packed))
        torch.cuda.synchronize()
        for x in ins:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                outs.append(ops.linear8(x, packed))
            graphs.append(g)
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(5):
        for t in outs:
            t.zero_()
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, want):
            assert torch.equal(a, b)


def test_gpu_refusals():
    x = _normal((4, 32), 1)
    w = _normal((8, 32), 2)
    with pytest.raises(TypeError):
        ops.linear8(x.float(), w)
    with pytest.raises(TypeError):
        ops.linear8(x.half(), w)
    with pytest.raises(ValueError):
        ops.linear8(x, w.cpu())
    with pytest.raises(ValueError):
        ops.swiglu8(x, x.cpu())
    with pytest.raises(ValueError):
        ops.rms_norm8(x, torch.ones(32))
    wide = torch.zeros(1, 16385, device="cuda")
    with pytest.raises(RuntimeError):
        ops.rms_norm8(wide, torch.ones(16385, device="cuda"))


def test_second_derivatives_are_refused():
    x = _normal((4, 32), 1).requires_grad_(True)
    w = _normal((8, 32), 2).requires_grad_(True)
    n = torch.ones(32, device="cuda", requires_grad=True)
    for y in (ops.linear8(x, w), ops.swiglu8(x, x), ops.rms_norm8(x, n)):
        with pytest.raises(RuntimeError, match="second derivative"):
            torch.autograd.grad(y.float().sum(), x, create_graph=True)


def test_gradients_of_shared_and_expanded_inputs():
    """The same tensor twice, a broadcast input, the same weight twice."""
    x = _normal((5, 200), 1).requires_grad_(True)
    ops.swiglu8(x, x).backward(torch.ones_like(x))
    (_, _), (dg, bg), (du, bu) = oracle.swiglu(
        x.detach(), x.detach(), torch.ones_like(x))
    # each part is rounded to bf16 before autograd adds them
    oracle.assert_within(x.grad, dg + du,
                         bg + bu + (dg.abs() + du.abs()) * 2.0 ** -8)
    row = _normal((1, 200), 2).requires_grad_(True)
    w = _normal((60, 200), 3, 0.1).requires_grad_(True)
    dy = _normal((7, 60), 4)
    wide = row.expand(7, 200)
    wide.retain_grad()
    y = ops.linear8(wide, w)
    y.backward(dy)
    want_y, want_dx, want_dw = oracle.linear(
        row.detach().expand(7, 200), [w.detach()], [dy])
    oracle.assert_within(y, *want_y[0])
    oracle.assert_within(wide.grad, *want_dx)
    oracle.assert_within(w.grad, *want_dw[0])
    # the same weight twice: both outputs are equal, the gradients add
    a, b = ops.linear8(row, w, w)
    assert torch.equal(a, b)
    ga, = torch.autograd.grad(a, w, dy[:1], retain_graph=False)
    assert ga.shape == w.shape


def test_weights_changed_before_backward_are_noticed():
    x = _normal((4, 32), 1).requires_grad_(True)
    w = _normal((8, 32), 2).requires_grad_(True)
    y = ops.linear8(x, w)
    with torch.no_grad():
        w.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.sum().backward()


# ------------------------------------------- every kernel, and large offsets
# Sizes that reach each tile size, K split for all tiles and for the last
# ones only, K shared by the waves, and few rows packed on the way; K short
# of one block, ending inside a quad of blocks, and long.
PLANS = [(1, 64, (48,)), (5, 700, (300, 20)), (16, 8, (16,)),
         (16, 2048, (8192,)), (13, 1000, (14000,)), (17, 300, (40,)),
         (32, 4096, (512,)), (48, 130, (1030,)), (64, 6000, (256,)),
         (100, 128, (5000,)), (129, 640, (2049,)), (256, 16384, (128,)),
         (700, 384, (700,)), (1025, 1024, (1025,)), (2048, 512, (2048, 700)),
         (3000, 200, (3000,)), (4200, 1536, (2500,)), (4352, 4096, (4352,)),
         (520, 12000, (390,)), (3001, 200, (2999,)), (2047, 512, (2701,)),
         (4617, 1792, (3457,)), (24, 512, (700, 60)), (32, 2048, (4100,)),
         (31, 1024, (8000,))]


@pytest.mark.parametrize("M,K,Ns", PLANS)
def test_linear8_over_its_kernels(M, K, Ns):
    x, ws, _ = _linear_inputs(M, K, Ns, seed=M + K)
    xq = oracle.held(x)
    with torch.no_grad():
        packed = ops.pack_weight8(*ws)
        for call in (ops.linear8(x, packed), ops.linear8(x, *ws)):
            call = call if isinstance(call, tuple) else (call,)
            for y, w in zip(call, ws):
                wq = oracle.held_weight(w)
                oracle.assert_within(y, xq @ wq.t(),
                                     oracle.product_bound(xq, wq))


@pytest.mark.parametrize("M,K", [(16, 3000), (32, 2000)])
def test_linear8_of_few_rows_holds_what_pack8_holds(M, K):
    """Rows packed on the way are rows packed before: the same codes, so
    results differ by the order of a sum only."""
    x, ws, _ = _linear_inputs(M, K, (200,))
    x[3, 100] = float("inf")
    x[M - 2, K - 1] = float("nan")
    x[5] = 0
    x[6, :] = 1e-39
    x[7, 5] = torch.finfo(torch.bfloat16).max
    xq, wq = oracle.held(x), oracle.held_weight(ws[0])
    with torch.no_grad():
        y = ops.linear8(x, ops.pack_weight8(ws[0]))
    bad = torch.zeros(M, dtype=torch.bool, device="cuda")
    bad[[3, M - 2]] = True
    assert y[bad].isnan().all()
    oracle.assert_within(y[~bad], (xq[~bad] @ wq.t()),
                         oracle.product_bound(xq[~bad], wq))


def test_one_dimensional_input():
    x, ws, _ = _linear_inputs(1, 200, (60, 50))
    with torch.no_grad():
        a, b = ops.linear8(x, *ws)
        c, d = ops.linear8(x[0], *ws)
        assert c.shape == (60,) and d.shape == (50,)
        assert torch.equal(a[0], c) and torch.equal(b[0], d)
        n = torch.ones(200, device="cuda")
        assert torch.equal(ops.rms_norm8(x[0], n), ops.rms_norm8(x, n)[0])
        assert torch.equal(ops.swiglu8(x[0], x[0]), ops.swiglu8(x, x)[0])
        assert torch.equal(ops.unpack8(ops.pack8(x[0])),
                           ops.unpack8(ops.pack8(x))[0])


def test_offsets_past_32_bits():
    R, C = 140001, 16384  # 2.3e9 values
    x = torch.empty(R, C, device="cuda", dtype=torch.bfloat16)
    x.normal_(generator=_gen(1))
    last = slice(R - 40, R)
    want = oracle.held(x[last])
    held = ops.pack8(x)
    assert torch.equal(ops.unpack8(held)[last].double(), want)
    del held
    # a product over all of it, and one with as large a result
    w = _normal((64, C), 2, 0.02)
    with torch.no_grad():
        y = ops.linear8(x, ops.pack_weight8(w))
    wq = oracle.held_weight(w)
    oracle.assert_within(y[last], want @ wq.t(),
                         oracle.product_bound(want, wq))
    narrow = x[:, :40]
    w = _normal((C, 40), 3, 0.1)
    with torch.no_grad():
        y = ops.linear8(narrow, ops.pack_weight8(w))
    xq, wq = oracle.held(narrow[last]), oracle.held_weight(w)
    oracle.assert_within(y[last], xq @ wq.t(), oracle.product_bound(xq, wq))
    del y
    # the norm and the gate, with their gradients
    n = torch.ones(C, device="cuda", requires_grad=True)
    x.requires_grad_(True)
    y = ops.rms_norm8(x, n)
    dx, _ = torch.autograd.grad(y, (x, n), x.detach())
    d = x.detach()[last]
    (wy, by), (wdx, bdx), _ = oracle.rms(d, n.detach(), d, 1e-5)
    oracle.assert_within(y[last], wy, by)
    oracle.assert_within(dx[last], wdx, bdx)
    del y, dx
    h = ops.swiglu8(x, x.detach())
    dg, = torch.autograd.grad(h, x, x.detach())
    (wh, bh), (wdg, bdg), _ = oracle.swiglu(d, d, d)
    oracle.assert_within(h[last], wh, bh)
    oracle.assert_within(dg[last], wdg, bdg)


# operands from 32 MB and results from 64 MB on pass by the caches
@pytest.mark.parametrize("R,C,dtype", [
    (9000, 4096, torch.bfloat16), (8191, 4104, torch.float16),
    (4100, 4096, torch.float32)])
def test_large_rows_pass_by_the_caches(R, C, dtype):
    x = _normal((R, C), 1, 2.0, dtype).requires_grad_(True)
    u = _normal((R, C), 2, 1.0, dtype).requires_grad_(True)
    w = (1 + 0.2 * _normal((C,), 3, dtype=torch.float32)).requires_grad_(True)
    d = _normal((R, C), 4, 1.0, dtype)
    got = ops.unpack8(ops.pack8(x))
    want = oracle.held(x.detach())
    assert torch.equal(got.double(), want.to(dtype).double())
    y = ops.rms_norm8(x, w)
    grads = torch.autograd.grad(y, (x, w), d)
    for got, (want, bound) in zip((y, *grads), oracle.rms(
            x.detach(), w.detach(), d, 1e-5)):
        oracle.assert_within(got, want, bound)
    h = ops.swiglu8(x, u)
    grads = torch.autograd.grad(h, (x, u), d)
    for got, (want, bound) in zip((h, *grads), oracle.swiglu(
            x.detach(), u.detach(), d)):
        oracle.assert_within(got, want, bound)


@pytest.mark.parametrize("M,K,Ns", [
    (4500, 4096, (128,)), (64, 4096, (4200,)), (9000, 200, (4096,)),
    (9001, 130, (4097,)), (300, 4097, (4101, 64))])
def test_large_operands_pass_by_the_caches(M, K, Ns):
    _check_linear(*_linear_inputs(M, K, Ns))


def test_a_batch_of_many_tokens_trains():
    """dW over a long axis: more K steps than a tile has rows."""
    x, ws, dys = _linear_inputs(40000, 130, (70,))
    _check_linear(x, ws, dys)


def test_a_graph_outlives_dropped_packed_weights():
    """A captured module call reads the weights that it was captured with."""
    m = ops.MaggyLinear8(512, 300).cuda().bfloat16()
    x = _normal((4, 512), 1)
    graph = torch.cuda.CUDAGraph()
    with torch.no_grad():
        ops.pack8_model(m)
        want = m(x)
        with torch.cuda.graph(graph):
            y = m(x)
    ops.drop8_model(m)
    junk = [torch.full((1 << 20,), 255, device="cuda", dtype=torch.uint8)
            for _ in range(16)]  # would land in freed memory
    for _ in range(3):
        y.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want)
    del junk
    assert len(m.group._captured) == 1
    ops.drop8_model(m, captured=True)
    assert not m.group._captured


def test_packed_weights_on_another_stream():
    """Packed behind long work on one stream, read at once on another; then
    dropped, and their memory offered for use, before that read runs."""
    m = ops.MaggyLinear8(2048, 2000).cuda().bfloat16()
    x = _normal((40, 2048), 1)
    big = torch.randn(4096, 4096, device="cuda")
    side = torch.cuda.Stream()
    with torch.no_grad():
        want = m(x)
        for _ in range(3):
            torch.cuda.synchronize()
            for _ in range(10):
                big @ big
            ops.pack8_model(m)
            with torch.cuda.stream(side):
                first = m(x)
                for _ in range(10):
                    big @ big
                second = m(x)
            sizes = [m.group.packed.codes.numel(),
                     m.group.packed.scales.numel()]
            ops.drop8_model(m)
            junk = [torch.full((n,), 255, device="cuda", dtype=torch.uint8)
                    for n in sizes for _ in range(4)]
            torch.cuda.synchronize()
            assert torch.equal(first, want) and torch.equal(second, want)
            del junk


def test_a_graph_takes_no_packed_weights_of_another_thread():
    """What generate packs for its call another thread does not read."""
    import threading

    m = ops.MaggyLinear8(512, 300).cuda().bfloat16()
    x = _normal((4, 512), 1)
    graph = torch.cuda.CUDAGraph()
    with torch.no_grad():
        m.group.pack(owner=threading.get_ident() + 1)
        want = m(x)
        with torch.cuda.graph(graph):
            y = m(x)
        assert not m.group._captured and m.group.packed is not None
        m.weight.mul_(2)
        graph.replay()  # packs the weights as they are now
        torch.cuda.synchronize()
        assert torch.equal(y, 2 * want)


def test_capture_beside_an_eager_graph_is_refused():
    """A leaf whose eager graph lives belongs to the default stream."""
    x = _normal((8, 256), 1)
    w = _normal((64, 256), 2, 0.1).requires_grad_(True)
    n = torch.ones(256, device="cuda", requires_grad=True)
    g = _normal((8, 256), 3).requires_grad_(True)
    for call, dy in ((lambda: ops.linear8(x, w), _normal((8, 64), 4)),
                     (lambda: ops.rms_norm8(x, n), _normal((8, 256), 5)),
                     (lambda: ops.swiglu8(g, x), _normal((8, 256), 6))):
        eager = call()
        torch.cuda.synchronize()
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            y = call()
            with pytest.raises(RuntimeError, match="eager graph"):
                y.backward(dy)
        eager.backward(dy)  # not hurt by it
        torch.cuda.synchronize()
    assert all(t.grad.isfinite().all() for t in (w, n, g))


def test_two_threads_at_once():
    """Forward and backward passes of two threads, each on its own stream."""
    from concurrent.futures import ThreadPoolExecutor

    def work(seed):
        x = _normal((300 + 50 * seed, 512), seed).requires_grad_(True)
        w1, w3 = [_normal((384, 512), seed + s, 0.05).requires_grad_(True)
                  for s in (10, 20)]
        n = torch.ones(512, device="cuda", requires_grad=True)
        h = ops.swiglu8(*ops.linear8(ops.rms_norm8(x, n), w1, w3))
        return [h.detach(), *torch.autograd.grad(
            h, [x, n, w1, w3], _normal(h.shape, seed + 30))]

    def on_stream(seed):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            out = [work(seed) for _ in range(10)]
        s.synchronize()
        return out

    want = [work(seed) for seed in (1, 2)]
    torch.cuda.synchronize()
    with ThreadPoolExecutor(2) as pool:
        got = list(pool.map(on_stream, (1, 2)))
    for outs, exact in zip(got, want):
        for out in outs:
            for a, b in zip(out, exact):
                assert torch.equal(a, b)


@pytest.mark.parametrize("how", ["again", "again, reentrant", "on the CPU"])
def test_what_is_kept_may_be_kept_elsewhere(how):
    """Recomputed in the backward pass, or held in host memory meanwhile."""
    from torch.utils.checkpoint import checkpoint

    norm = ops.MaggyRMSNorm8(256).cuda()
    ff = ops.MaggyFeedForward8(256, 384).cuda().bfloat16()
    x = _normal((70, 256), 1).requires_grad_(True)
    dy = _normal((70, 256), 2)
    params = [x, *norm.parameters(), *ff.parameters()]

    def grads(y):
        for p in params:
            p.grad = None
        y.backward(dy)
        return [p.grad for p in params]

    want = grads(ff(norm(x)))
    if how == "on the CPU":
        with torch.autograd.graph.save_on_cpu():
            y = ff(norm(x))
    else:
        y = checkpoint(lambda x: ff(norm(x)), x,
                       use_reentrant="reentrant" in how)
    for a, b in zip(grads(y), want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("wtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("kind", ["FusedAdam", "FusedSGD"])
def test_packed_weights_that_the_optimizer_updates(kind, wtype):
    """Packed between the gradients and the step, whose kernels write."""
    m = torch.nn.Sequential(*[ops.MaggyLinear8(256, 256) for _ in range(2)])
    m = m.cuda().to(wtype)
    other = ops.MaggyLinear8(256, 256).cuda().bfloat16()
    x = _normal((4, 256), 1)
    opt = getattr(ops, kind)(m.parameters(), lr=0.1)
    m(x).float().square().sum().backward()
    ops.pack8_model(m)
    ops.pack8_model(other)
    with torch.no_grad():
        before = m(x)
        opt.step()
        got = m(x)
        want = ops.linear8(ops.linear8(x, m[0].weight), m[1].weight)
    assert torch.equal(got, want) and not torch.equal(got, before)
    assert other.group.packed is not None  # not of this optimizer


@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_is_refused(grad):
    from torch.autograd import forward_ad

    from tests.test_block8 import _forward_mode_calls

    x, w = _normal((4, 32), 1), _normal((8, 32), 2)
    n = torch.ones(32, device="cuda")
    with torch.set_grad_enabled(grad), forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        for i, call in enumerate(_forward_mode_calls(x, w, n)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call(dual)
                print("not refused:", i)
            call(x)
        with pytest.raises(RuntimeError, match="forward-mode"):
            ops.linear8(x, forward_ad.make_dual(w, torch.ones_like(w)))
        with pytest.raises(RuntimeError, match="forward-mode"):
            ops.rms_norm8(x, forward_ad.make_dual(n, torch.ones_like(n)))


# M rows, so that the weights' gradients sum over M; N and K make every tile
# size, with K split and not, and tiles that reach over two weights
@pytest.mark.parametrize("M,K,Ns", [
    (70, 130, (60, 50)), (150, 300, (129, 1, 77)), (600, 1024, (700, 500)),
    (2048, 1030, (300, 1000)), (4096, 256, (130, 129, 128, 127)),
    (300, 4000, (2600, 1500)), (6000, 4096, (4100, 200))])
@pytest.mark.parametrize("wtype", [torch.bfloat16, torch.float32])
def test_gradients_of_several_weights_are_tensors_of_their_own(M, K, Ns,
                                                               wtype):
    x, ws, dys = _linear_inputs(M, K, Ns, wtype)
    ws = [w.requires_grad_(True) for w in ws]
    dws = torch.autograd.grad(ops.linear8(x, *ws), ws, dys)
    _, _, want = oracle.linear(x, [w.detach() for w in ws], dys)
    for i, (d, (exact, bound)) in enumerate(zip(dws, want)):
        assert d.shape == ws[i].shape and d.is_contiguous()
        oracle.assert_within(d, exact, bound, "dw{}".format(i))
        size = d.untyped_storage().nbytes()
        assert d.storage_offset() == 0
        assert size == d.numel() * d.element_size()
    assert len({d.untyped_storage().data_ptr() for d in dws}) == len(dws)


# M, K and rows of the weights, so that dW takes: 256 x 256, 128 x 256,
# 128 x 128 and 64 x 64 tiles, each whole and with K split and joined
@pytest.mark.parametrize("M,K,Ns", [
    (300, 3001, (60, 2500, 60)), (6000, 3001, (2500, 2500, 1500)),
    (300, 3001, (300, 700, 129)), (6000, 3001, (129, 1000, 1500)),
    (300, 130, (1500, 60, 2500)), (12000, 130, (300, 129)),
    (300, 130, (700, 60, 129)), (6000, 130, (60,))])
def test_gradients_of_fp32_weights_over_the_kernels(M, K, Ns):
    _check_linear(*_linear_inputs(M, K, Ns, torch.float32))


def test_a_refused_launch_is_reported_and_not_left_behind():
    """A grid of no workgroups, which the runtime refuses."""
    from tests.test_block8 import _launchers

    lib, names, call = _launchers()
    torch.cuda.synchronize()
    lib.hipGetLastError()
    for name in names:
        assert call(name, 0) != 0, name
        assert lib.hipGetLastError() == 0, name
    torch.cuda.synchronize()


def test_capture_beside_an_eager_graph_is_refused_behind_views():
    """Leaves that a call reshapes or converts before its kernels."""
    x = _normal((2, 4, 256), 1).requires_grad_(True)
    w = _normal((64, 256), 2, 0.1)
    n = torch.ones(256, device="cuda", dtype=torch.bfloat16,
                   requires_grad=True)
    far = _normal((4, 2, 256), 3).requires_grad_(True)
    wide = _normal((8, 256), 4, dtype=torch.float32).requires_grad_(True)
    for call, leaf, shape in (
            (lambda: ops.linear8(x, w), x, (2, 4, 64)),
            (lambda: ops.rms_norm8(x.detach(), n), n, (2, 4, 256)),
            (lambda: ops.swiglu8(x, x.detach()), x, (2, 4, 256)),
            (lambda: ops.linear8(far.transpose(0, 1)[..., :], w), far,
             (2, 4, 64)),
            (lambda: ops.linear8(wide.bfloat16(), w), wide, (8, 64))):
        dy = _normal(shape, 5)
        eager = call()
        torch.cuda.synchronize()
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            y = call()
            with pytest.raises(RuntimeError, match="eager graph"):
                y.backward(dy)
        eager.backward(dy)  # not hurt by it
        torch.cuda.synchronize()
        assert leaf.grad.isfinite().all()


def test_negative_views():
    """Tensors whose sign is a bit of the tensor, as the imaginary part of a
    conjugate has it."""
    neg = torch._neg_view
    x, w = _normal((5, 200), 1), _normal((60, 200), 2, 0.1)
    n, dy = torch.randn(200, device="cuda"), _normal((5, 200), 3)
    assert neg(x).is_neg()
    assert torch.equal(ops.unpack8(ops.pack8(neg(x))),
                       ops.unpack8(ops.pack8(-x)))
    for grad in (False, True):
        x = x.detach().requires_grad_(grad)
        for a, b in ((ops.linear8(neg(x), neg(w)), ops.linear8(-x, -w)),
                     (ops.swiglu8(neg(x), neg(dy)), ops.swiglu8(-x, -dy)),
                     (ops.rms_norm8(neg(x), neg(n)), ops.rms_norm8(-x, -n))):
            assert torch.equal(a, b)
            if grad:
                d = torch.randn_like(a)
                da, = torch.autograd.grad(a, x, neg(d), retain_graph=True)
                db, = torch.autograd.grad(b, x, -d, retain_graph=True)
                assert torch.equal(da, db)
    z = torch.randn(7, 1, device="cuda", dtype=torch.complex64)
    part = z.conj().imag
    assert part.is_neg()
    assert torch.equal(ops.unpack8(ops.pack8(part)),
                       ops.unpack8(ops.pack8(-z.imag.clone())))


def test_gradients_past_32_bits_of_several_weights():
    """The second weight's rows lie beyond 2^31 values of the product."""
    M, K, Ns = 70, 16384, (139990, 300)
    x = _normal((M, K), 1)
    ws = [torch.empty(n, K, device="cuda", dtype=torch.bfloat16)
          .normal_(0.0, 0.02, generator=_gen(2 + i)).requires_grad_(True)
          for i, n in enumerate(Ns)]
    dys = [_normal((M, n), 5 + i, 1e-3) for i, n in enumerate(Ns)]
    ys = ops.linear8(x, *ws)
    dws = torch.autograd.grad(ys, ws, dys)
    for y, dw, w, dy in zip(ys, dws, ws, dys):
        for rows in (slice(0, 40), slice(w.shape[0] - 40, w.shape[0])):
            # whole blocks of 128 rows, as the weights are packed
            lo = rows.start // 128 * 128
            wq = oracle.held_weight(w.detach()[lo:rows.stop])
            xq = oracle.held(x)
            skip = rows.start - lo
            oracle.assert_within(y[:, rows], xq @ wq[skip:].t(),
                                 oracle.product_bound(xq, wq[skip:]))
            _, _, ((want, bound),) = oracle.linear(
                x, [w.detach()[rows]], [dy[:, rows]])
            oracle.assert_within(dw[rows], want, bound)


@torch.no_grad()
def test_ablated_and_hooked_layers_decode():
    from maggy_amd.ablation.ablationstudy import drop_layers

    m = _llama().eval()
    tokens = torch.randint(0, 256, (2, 8), device="cuda")
    before, seen = m(tokens), []
    drop_layers(m, "layers.0.attn.wo")
    hook = m.layers[1].ffn.w3.register_forward_hook(
        lambda mod, args, out: seen.append(out))
    for _ in range(2):
        logits = m(tokens)
        assert not torch.equal(logits, before)
        out = m.generate(tokens, 5)
        assert seen and seen[0].dtype == torch.bfloat16
        ops.pack8_model(m)
        assert torch.equal(m(tokens), logits)
        assert torch.equal(m.generate(tokens, 5), out)
    hook.remove()
    seen.clear()
    ops.drop8_model(m)
    logits = m(tokens)
    ops.pack8_model(m)
    assert torch.equal(m(tokens), logits) and not seen
