"""The layer's operators as they are used together (`NSABlock`: training, prefill, decoding), and the circumstances a program
brings: other streams, two calls at once, captured graphs, views off the 16-byte grid, operands in other layouts."""
import subprocess
import sys
import textwrap

import pytest
import torch

pytestmark = pytest.mark.gpu

BF = 2.0 ** -8            # one rounding to bf16, relative


@pytest.fixture(scope="module")
def nsa():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import nsa_from_scratch_b200 as m
    return m


def randn(*shape, seed=0, std=1.0, dtype=torch.bfloat16):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * std).to(dtype).cuda()


def rel(a, b):
    return float((a.double() - b.double()).norm() / b.double().norm())


def make_block(nsa, hidden=192, H=4, Hkv=2, D=64, F=344, sections=(8, 12, 12), seed=0, top_k=8):
    """Every block that a row may see is listed, so that no rounding decides a selection."""
    cfg = nsa.NSAConfig(block_size_c=32, stride_c=16, top_k=top_k, window_size=96, select_per_group=True)
    torch.manual_seed(seed)
    block = nsa.NSABlock(hidden, H, D, cfg, F, n_kv_heads=Hkv, rope_sections=sections)
    with torch.no_grad():
        for p in (block.attn_norm, block.mlp_norm):
            p.add_(0.2 * torch.randn_like(p))
    return block.to(device="cuda", dtype=torch.bfloat16)


def video_positions(B, T, start=1000):
    at = torch.arange(T, device="cuda")
    return torch.stack([at // 24, at // 6 % 4, at % 6]).add(start)[:, None].expand(3, B, T).contiguous()


def plain_block(nsa, block, x, pos):
    """The block's formulas in 64 bits around the framework's own attention (whose operands are 16-bit)."""
    a, D = block.attn, block.attn.head_dim
    B, T, _ = x.shape

    def norm(t, w):
        return t * (t.square().mean(-1, keepdim=True) + block.eps).rsqrt() * w.double()

    axis = [i for i, n in enumerate(block.rope_sections) for _ in range(n)]
    inv = nsa.rope_frequencies(D, block.rope_base)
    ang = torch.stack([pos[i].double() * inv[j] for j, i in enumerate(axis)], -1)[:, None]

    def turn(t):
        p, q = t.chunk(2, -1)
        return torch.cat((p * ang.cos() - q * ang.sin(), q * ang.cos() + p * ang.sin()), -1)

    h = norm(x, block.attn_norm)
    q, k, v = ((h @ m.weight.double().T).view(B, T, -1, D).transpose(1, 2) for m in (a.q_proj, a.k_proj, a.v_proj))
    gates = (h @ a.gate.weight.double().T).view(B, T, a.n_heads, 3).permute(0, 2, 1, 3)
    out = nsa.nsa_forward(*(t.to(torch.bfloat16).contiguous() for t in (turn(q), turn(k), v)), a.nsa_cfg, gate_logits=gates.to(torch.bfloat16).contiguous())
    x = x + out.double().transpose(1, 2).reshape(B, T, -1) @ a.o_proj.weight.double().T
    h = norm(x, block.mlp_norm)
    g = h @ block.gate_proj.weight.double().T
    return x + (g * torch.sigmoid(g) * (h @ block.up_proj.weight.double().T)) @ block.down_proj.weight.double().T


@pytest.mark.parametrize("B,T", [(1, 256), (2, 300), (1, 65)])
def test_block_training_step(nsa, B, T):
    """Result and every gradient.  A value passes about a dozen roundings to bf16 on its way through the block, and about
    twice that on the way back; each is off by at most 2^-8 of its size."""
    block = make_block(nsa)
    x = randn(B, T, 192, seed=1).requires_grad_(True)
    pos = video_positions(B, T)
    dy = randn(B, T, 192, seed=2)
    y = block(x, pos)
    params = list(block.parameters())
    grads = torch.autograd.grad(y, [x, *params], dy)
    xd = x.detach().double().requires_grad_(True)
    ref = plain_block(nsa, block, xd, pos)
    want = torch.autograd.grad(ref, [xd, *params], dy.double())
    assert rel(y.detach(), ref.detach()) <= 12 * BF
    for g, r, (name, p) in zip(grads, want, [("x", x), *block.named_parameters()]):
        assert g.shape == p.shape and g.dtype == p.dtype and rel(g, r) <= 24 * BF, (name, rel(g, r))
    with torch.no_grad():                                        # prefill: the inference route of the attention
        assert rel(block(x, pos), ref.detach()) <= 12 * BF


def test_block_decoding_equals_prefill(nsa):
    """Positions fed a chunk, then one or two at a time, against the whole sequence at once."""
    block = make_block(nsa, sections=None, seed=3)
    B, T = 2, 150
    x = randn(B, T, 192, seed=4)
    with torch.no_grad():
        whole = block(x)
        cache = block.new_cache(B, 192)
        parts = [block(x[:, :100].contiguous(), cache=cache)]
        t = 100
        while t < T:
            n = 1 if t % 3 else 2
            n = min(n, T - t)
            parts.append(block(x[:, t:t + n].contiguous(), cache=cache))
            t += n
    assert cache.length == T
    got = torch.cat(parts, 1)
    assert rel(got, whole) <= 24 * BF
    assert rel(got[:, 100:], whole[:, 100:]) <= 24 * BF
    with pytest.raises(RuntimeError, match="no gradients"):
        block(x[:, :1].contiguous().requires_grad_(True), cache=cache)
    with pytest.raises(ValueError, match="need positions"):
        make_block(nsa)(x)


def test_attend_with_residual(nsa):
    """The residual in the output projection's epilogue: the same sum, rounded once."""
    block = make_block(nsa, sections=None)
    x, r = randn(1, 130, 192, seed=5), randn(1, 130, 192, seed=6)
    pos = torch.arange(130, device="cuda")[None, None]
    with torch.no_grad():
        a = block.attn.attend(x, pos, nsa.rope_frequencies(64), (32,))
        b = block.attn.attend(x, pos, nsa.rope_frequencies(64), (32,), residual=r)
    want = a.double() + r.double()
    assert float(((b.double() - want).abs() - BF * (a.double().abs() + want.abs())).max()) <= 0


def test_fp8_projection_behind_the_norm(nsa):
    """rms_norm_fp8 -> linear_fp8 against the 64-bit norm and product: two roundings to e4m3 (2^-4 each), one to bf16."""
    x, r, w = randn(70, 1024, seed=1), randn(70, 1024, seed=2, std=2.0), randn(1024, seed=3)
    weight = randn(520, 1024, seed=4, std=1 / 32)
    q, s, h = nsa.rms_norm_fp8(x, w, residual=r)
    w8, ws = nsa.quantize_rows_to_fp8(weight)
    y = nsa.linear_fp8(q, w8, s, ws)
    hd = h.double()
    n = hd * (hd.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * w.double()
    assert rel(y, n @ weight.double().T) <= 2 * 2.0 ** -4 + BF


def everything(nsa, x, w, sq, dy):
    """One training step through every operator, gradients of x, w and sq."""
    y, h = nsa.rms_norm(x, w, residual=x)
    z = nsa.linear(y, sq, w, activation="gelu_tanh", residual=h)
    o = nsa.gated_mlp(z, sq, sq, sq, residual=z)
    q = o.view(1, -1, 4, 64)
    pos = torch.arange(q.shape[1], device=x.device).view(1, 1, -1)
    t = nsa.rope_axes_to_heads(q, q, q, pos, nsa.rope_frequencies(64, device=x.device), (32,))
    out = t[0] + t[1] + t[2]
    return (out, *torch.autograd.grad(out, (x, w, sq), dy))


def step_inputs(rows, seed):
    x, w, sq = (randn(*s, seed=seed + i, std=v).requires_grad_(True) for i, (s, v) in enumerate((((rows, 256), 1.0), ((256,), 1.0), ((256, 256), 1 / 16))))
    return x, w, sq, randn(1, 4, rows, 64, seed=seed + 9)


@pytest.mark.parametrize("rows", [3, 40, 300])
def test_other_streams_and_two_calls_at_once(nsa, rows):
    a, b = step_inputs(rows, 0), step_inputs(rows, 50)
    want = [[t.clone() for t in everything(nsa, *s)] for s in (a, b)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(4):
        for i, s in enumerate((a, b)):
            streams[i].wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(streams[i]):
                got[i] = everything(nsa, *s)
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert all(torch.equal(p, q) for p, q in zip(g, w))


@pytest.mark.parametrize("rows", [3, 300])
def test_captured_step_replays_with_new_inputs(nsa, rows):
    """Forward and backward in one CUDA graph."""
    x, w, sq, dy = step_inputs(rows, 0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            everything(nsa, x, w, sq, dy)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = everything(nsa, x, w, sq, dy)
    for seed in (100, 200):
        new = step_inputs(rows, seed)
        with torch.no_grad():
            for old, n in zip((x, w, sq, dy), new):
                old.copy_(n)
        graph.replay()
        torch.cuda.synchronize()
        for g, r in zip(out, everything(nsa, *new)):
            assert torch.equal(g, r)


def test_two_captured_graphs_do_not_share_scratch(nsa):
    steps = [step_inputs(rows, rows) for rows in (200, 130)]
    graphs, outs = [], []
    for s in steps:
        everything(nsa, *s)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(everything(nsa, *s))
        graphs.append(g)
    want = [[t.clone() for t in everything(nsa, *s)] for s in steps]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(3):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for o, w in zip(outs, want):
        assert all(torch.equal(p, q) for p, q in zip(o, w))


def off_grid(t):
    """The same values, dense, one element behind a 16-byte boundary."""
    buf = torch.empty(t.numel() + 1, device=t.device, dtype=t.dtype)
    return buf[1:].view(t.shape).copy_(t.detach())


@pytest.mark.parametrize("M", [5, 20, 140])
def test_operands_off_the_16_byte_grid(nsa, M):
    """Views that start anywhere: the same results to the order of the sums, gradients included."""
    x, w, b, r, dy = randn(M, 136, seed=1), randn(72, 136, seed=2, std=0.1), randn(72, seed=3), randn(M, 72, seed=4), randn(M, 72, seed=5)

    def step(x, w, b, r, dy):
        ls = [t.detach().requires_grad_(True) for t in (x, w, b, r)]
        y = nsa.linear(*ls[:3], activation="silu", residual=ls[3])
        return (y.detach(), *torch.autograd.grad(y, ls, dy))

    for p, q in zip(step(*(off_grid(t) for t in (x, w, b, r, dy))), step(x, w, b, r, dy)):
        assert rel(p, q) <= 2 * BF
    m = [randn(*s, seed=6 + i, std=0.1) for i, s in enumerate(((200, 136), (200, 136), (136, 200)))]

    def mlp(x, *m):
        ls = [t.detach().requires_grad_(True) for t in (x, *m)]
        y = nsa.gated_mlp(*ls)
        return (y.detach(), *torch.autograd.grad(y, ls, x.detach()))

    for p, q in zip(mlp(*(off_grid(t) for t in (x, *m))), mlp(x, *m)):
        assert rel(p, q) <= 4 * BF
    for dt in (torch.bfloat16, torch.float32):
        a, c, g = x.to(dt), randn(136, seed=11, dtype=dt), x.to(dt)

        def norm(a, c, g):
            ls = [t.detach().requires_grad_(True) for t in (a, c)]
            y, h = nsa.rms_norm(ls[0], ls[1], residual=a)
            return (y.detach(), h.detach(), *torch.autograd.grad((y, h), ls, (g, g)))

        for p, q in zip(norm(*(off_grid(t) for t in (a, c, g))), norm(a, c, g)):
            assert rel(p, q) <= BF
    x8, xs = nsa.quantize_rows_to_fp8(x)
    w8, ws = nsa.quantize_rows_to_fp8(w)
    buf = torch.empty(x8.numel() + 1, device="cuda", dtype=torch.uint8)
    shifted = buf[1:].copy_(x8.view(torch.uint8).view(-1)).view(torch.float8_e4m3fn).view(x8.shape)
    assert rel(nsa.linear_fp8(shifted, w8, off_grid(xs), off_grid(ws)), nsa.linear_fp8(x8, w8, xs, ws)) <= 2 * BF
    q8, s8 = nsa.quantize_rows_to_fp8(off_grid(x))
    assert torch.equal(q8.view(torch.uint8), x8.view(torch.uint8)) and torch.equal(s8, xs)
    q = randn(1, M, 2, 64, seed=13)
    pos = torch.arange(M, device="cuda").view(1, 1, M)
    inv = nsa.rope_frequencies(64)
    for p, t in zip(nsa.rope_axes_to_heads(off_grid(q), off_grid(q), off_grid(q), pos, inv, (32,)), nsa.rope_axes_to_heads(q, q, q, pos, inv, (32,))):
        assert torch.equal(p, t)


def test_layouts_other_than_dense(nsa):
    """Transposed, expanded and sliced operands give what their dense copies give; strict layout checking refuses them."""
    from nsa_from_scratch_b200 import ops
    x, w = randn(64, 48, seed=1).T, randn(64, 40, seed=2).T
    r = randn(40, seed=3).expand(48, 40)
    assert torch.equal(nsa.linear(x, w, residual=r), nsa.linear(x.contiguous(), w.contiguous(), residual=r.contiguous()))
    assert torch.equal(nsa.rms_norm(x, w[0]), nsa.rms_norm(x.contiguous(), w[0].contiguous()))
    three = randn(2, 3, 5, 64, seed=4)                               # leading dimensions stay
    assert nsa.linear(three, w.contiguous()).shape == (2, 3, 5, 40) and nsa.rms_norm(three, w[0].contiguous()).shape == three.shape
    assert torch.equal(nsa.linear(three, w.contiguous()).view(30, 40), nsa.linear(three.view(30, 64), w.contiguous()))
    row = randn(64, seed=5)
    assert torch.equal(nsa.linear(row, w.contiguous())[None], nsa.linear(row[None], w.contiguous()))
    ops.set_strict_layout(True)
    try:
        with pytest.raises(ValueError, match="not contiguous"):
            nsa.linear(x, w)
        leaf = x.contiguous().requires_grad_(True)
        nsa.linear(leaf, w.contiguous()).sum().backward()            # autograd's own expanded gradient is no caller's layout
        assert leaf.grad is not None
    finally:
        ops.set_strict_layout(False)


def test_shared_weights_and_repeated_inputs(nsa):
    """The same tensor in several places: its gradient is the sum over them."""
    x, s = randn(40, 64, seed=1), randn(64, 64, seed=2, std=1 / 8)
    a = s.clone().requires_grad_(True)
    three = [s.clone().requires_grad_(True) for _ in range(3)]
    dy = randn(40, 64, seed=3)
    g, = torch.autograd.grad(nsa.gated_mlp(x, a, a, a), a, dy)
    gs = torch.autograd.grad(nsa.gated_mlp(x, *three), three, dy)
    assert rel(g, sum(t.double() for t in gs)) <= 2 * BF
    leaf = x.clone().requires_grad_(True)
    g, = torch.autograd.grad(nsa.linear(leaf, s, residual=leaf), leaf, dy)
    assert rel(g, dy.double() @ s.double() + dy.double()) <= 2 * BF


def test_no_second_differentiation(nsa):
    x, s = randn(8, 64, seed=1).requires_grad_(True), randn(64, 64, seed=2)
    g, = torch.autograd.grad(nsa.linear(x, s, activation="silu").square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.sum().backward()


def test_no_second_differentiation_of_any(nsa):
    x, s, w = randn(8, 64, seed=1).requires_grad_(True), randn(64, 64, seed=2), randn(64, seed=3)
    q = randn(1, 8, 2, 64, seed=4).requires_grad_(True)
    pos, inv = torch.arange(8, device="cuda").view(1, 1, 8), nsa.rope_frequencies(64)
    for leaf, out in ((x, lambda: nsa.rms_norm(x, w)), (x, lambda: nsa.rms_norm(x, w, residual=x)[0]), (x, lambda: nsa.gated_mlp(x, s, s, s)),
                      (q, lambda: nsa.rope_axes_to_heads(q, q, q, pos, inv, (32,))[1])):
        g, = torch.autograd.grad(out().float().square().sum(), leaf, create_graph=True)
        with pytest.raises(RuntimeError, match="once_differentiable"):
            g.sum().backward()


def test_only_the_gradients_asked_for(nsa):
    """torch.autograd.grad for some of the inputs: the same values, and no memory for the others' gradients."""
    x, dy = randn(48, 64, seed=1).requires_grad_(True), randn(48, 4096, seed=2)
    w, b = randn(4096, 64, seed=3).requires_grad_(True), randn(4096, seed=4).requires_grad_(True)
    wg, wu, wd = (randn(4096, 64, seed=5 + i).requires_grad_(True) for i in range(3))
    wd = wd.detach().T.contiguous().requires_grad_(True)
    for y, leaves, d in ((nsa.linear(x, w, b), (x, w, b), dy), (nsa.gated_mlp(x, wg, wu, wd), (x, wg, wu, wd), randn(48, 64, seed=9))):
        every = torch.autograd.grad(y, leaves, d, retain_graph=True)
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        torch.autograd.grad(y, leaves, d, retain_graph=True)
        most = torch.cuda.max_memory_allocated() - before
        for leaf, want in zip(leaves, every):
            torch.cuda.reset_peak_memory_stats()
            got, = torch.autograd.grad(y, leaf, d, retain_graph=True)
            assert torch.equal(got, want)
            assert torch.cuda.max_memory_allocated() - before < most


def test_block_first_used_in_inference_mode_then_trained(nsa):
    blk = nsa.NSABlock(64, 2, 64, nsa.NSAConfig(block_size_c=64, top_k=2, window_size=64), 96, n_kv_heads=1).cuda().bfloat16()
    x = randn(1, 70, 64, seed=1)
    with torch.inference_mode():
        first = blk(x)
    blk(x).float().square().mean().backward()
    assert blk.gate_proj.weight.grad is not None and torch.equal(blk(x).detach(), blk(x).detach())
    assert torch.isfinite(first).all()


def test_block_first_used_in_a_capture(nsa):
    """A block whose first call is captured: what it makes for itself there is filled at replay, and is no eager call's."""
    cfg = nsa.NSAConfig(block_size_c=64, top_k=2, window_size=64)
    blk = nsa.NSABlock(64, 2, 64, cfg, 96, n_kv_heads=1).cuda().bfloat16()
    twin = nsa.NSABlock(64, 2, 64, cfg, 96, n_kv_heads=1).cuda().bfloat16()
    twin.load_state_dict(blk.state_dict())
    x = randn(1, 70, 64, seed=1)
    pos = torch.arange(70, device="cuda").view(1, 1, 70)
    with torch.no_grad():
        want = twin(x, pos)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = blk(x, pos)
        assert torch.equal(blk(x, pos), want)              # before any replay
        g.replay()
        assert torch.equal(y, want)


def test_first_calls_of_a_process_captured(nsa):
    """Nothing that an operator sets up for itself on its first call stands in the way of a capture."""
    code = textwrap.dedent("""
        import torch, nsa_from_scratch_b200 as nsa
        torch.manual_seed(0)
        bf = dict(device="cuda", dtype=torch.bfloat16)
        x, few, w, norm = torch.randn(256, 512, **bf), torch.randn(8, 512, **bf), torch.randn(512, 512, **bf) / 24, torch.ones(512, **bf)
        wg, wu, wd = torch.randn(1408, 512, **bf) / 24, torch.randn(1408, 512, **bf) / 24, torch.randn(512, 1408, **bf) / 38
        q, pos, inv = torch.randn(2, 128, 4, 64, **bf), torch.arange(128, device="cuda").repeat(1, 2, 1), nsa.rope_frequencies(64)
        torch.cuda.synchronize()
        def run():
            h, r = nsa.rms_norm(x, norm, residual=x)
            a = nsa.linear(h, w, residual=r)
            (e, es), (k, ks) = nsa.rms_norm_fp8(x, norm), nsa.quantize_rows_to_fp8(w)
            return (a, nsa.gated_mlp(a, wg, wu, wd, residual=a), nsa.linear(few, w), nsa.gated_mlp(few, wg, wu, wd), nsa.linear_fp8(e, k, es, ks),
                    *nsa.rope_axes_to_heads(q, q, q, pos, inv, (32,)))
        with torch.no_grad():
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                got = run()
            g.replay()
            torch.cuda.synchronize()
            print("SAME", all(torch.equal(a, b) for a, b in zip(got, run())))
    """)
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300, cwd=__file__.rsplit("/tests/", 1)[0])
    assert r.returncode == 0 and "SAME True" in r.stdout, (r.returncode, r.stdout[-500:], r.stderr[-1500:])


def test_status_word_of_the_products(nsa):
    from nsa_from_scratch_b200 import _lib as L, ops
    lib = L.load()
    ops.device_status()
    L.check(lib.nsa_debug_set_device_status(4, 3), "set")
    with pytest.raises(RuntimeError, match="gave up waiting"):
        ops.device_status()
    ops.device_status()


@pytest.mark.parametrize("way", ["backward", "grad"])
def test_backward_captured_beside_a_live_eager_graph(nsa, way):
    """An eager graph of the same leaves lives while forward and backward are captured.  torch ties the leaves' gradient nodes
    to the eager stream then and refuses the capture (for its own operators alike); what matters is that the process gets
    an answer, right gradients or an exception, and goes on: it runs in a process of its own."""
    code = textwrap.dedent("""
        import torch, nsa_from_scratch_b200 as nsa
        torch.manual_seed(0)
        x = torch.randn(300, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
        w = torch.randn(64, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
        def step():
            loss = nsa.gated_mlp(nsa.linear(x, w), w, w, w).float().square().mean()
            if WAY == "grad":
                return torch.autograd.grad(loss, (x, w))
            x.grad = w.grad = None
            loss.backward()
            return x.grad, w.grad
        want = [t.clone() for t in step()]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        eager = nsa.gated_mlp(nsa.linear(x, w), w, w, w).float().square().mean()
        try:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                got = step()
            g.replay()
            torch.cuda.synchronize()
            print("CAPTURED", all(torch.equal(a, b) for a, b in zip(got, want)))
        except RuntimeError as e:
            print("REFUSED", str(e)[:80])
        again = torch.autograd.grad(eager, (x, w))
        torch.cuda.synchronize()
        print("AFTERWARDS", all(torch.equal(a, b) for a, b in zip(again, want)))
    """).replace("WAY", repr(way))
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300, cwd=__file__.rsplit("/tests/", 1)[0])
    assert r.returncode == 0 and "AFTERWARDS True" in r.stdout, (r.returncode, r.stdout[-500:], r.stderr[-1500:])
    assert "CAPTURED True" in r.stdout or "REFUSED" in r.stdout, r.stdout[-500:]
