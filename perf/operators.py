"""The operators around the attention of a decoder layer, as measurable cases.

Kinds (`case["kind"]`):

  norm     root-mean-square norm behind the residual's addition: 16-bit result, fp8 result with a scale per row, and
           the gradients of a training step
  rope     rotary embedding whose frequencies are dealt out to several position axes (time, height, width), from the
           projections' token-major tensors to the attention's head-major ones, and its gradients
  linear   matrix product with bias, activation and residual in its epilogue: 16-bit operands, fp8 operands with scales
           per row of both, and the gradients of a training step
  ffn      gated feed-forward block: down(act(gate(x)) * up(x)) (+ residual), and the gradients of a training step

Feature sizes are those of this repository's models: hidden sizes are heads * head size (12 x 64, 16 x 64, 64 x 64,
64 x 128), projections add the KV heads; gated blocks are about 8/3 as wide as the hidden size, as their kind is.
"""
import math

import torch

own = False

EPS = 1e-6
BASE = 10000.0
E4M3_MAX = 448.0
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32, "e4m3": torch.float8_e4m3fn}


# ---------------------------------------------------------------- cases

def listed():
    return [
        # One decoding step of eight conversations: launches and latency count.
        {"name": "norm_decode_b8", "kind": "norm", "mode": "fwd", "rows": 8, "hidden": 4096, "dtype": "bf16", "wdtype": "bf16", "residual": True},
        # Prefill in front of fp8 projections, the widest hidden size.
        {"name": "norm_fp8_16k", "kind": "norm", "mode": "fp8", "rows": 16384, "hidden": 8192, "dtype": "bf16", "wdtype": "bf16", "residual": True},
        # Training on a ragged batch, fp16 activations beside fp32 norm weights.
        {"name": "norm_train_ragged", "kind": "norm", "mode": "train", "rows": 8189, "hidden": 4096, "dtype": "fp16", "wdtype": "fp32", "residual": True},
        # One new token of each of eight long conversations.
        {"name": "rope_decode_b8", "kind": "rope", "mode": "fwd", "B": 8, "T": 1, "H": 64, "Hkv": 4, "D": 128, "sections": "16,24,24", "dtype": "bf16", "far": 60000},
        # Prefill of a video's patches behind a long text, q, k and v as slices of one packed projection.
        {"name": "rope_video_32k", "kind": "rope", "mode": "fwd", "B": 1, "T": 32768, "H": 64, "Hkv": 4, "D": 128, "sections": "16,24,24", "dtype": "bf16", "far": 250000},
        # Training at the training model's heads, fp32 projections, an odd length.
        {"name": "rope_train_odd", "kind": "rope", "mode": "train", "B": 2, "T": 4001, "H": 12, "Hkv": 1, "D": 64, "sections": "8,12,12", "dtype": "fp32", "far": 5000},
        # The output projection of one decoding step, residual in the epilogue: the weights' bytes count.
        {"name": "linear_decode_b8", "kind": "linear", "mode": "fwd", "M": 8, "K": 8192, "N": 8192, "dtype": "bf16", "bias": False, "act": "", "residual": True},
        # The fused q, k and v projection of a prefill on fp8 operands.
        {"name": "linear_fp8_8k", "kind": "linear", "mode": "fwd", "M": 8192, "K": 8192, "N": 9216, "dtype": "e4m3", "bias": True, "act": "", "residual": False},
        # Training of a biased projection with an activation, an odd number of tokens.
        {"name": "linear_train_odd", "kind": "linear", "mode": "train", "M": 4001, "K": 4096, "N": 4096, "dtype": "bf16", "bias": True, "act": "gelu_tanh", "residual": True},
        # The feed-forward block of one decoding step.
        {"name": "ffn_decode_b4", "kind": "ffn", "mode": "fwd", "M": 4, "hidden": 4096, "F": 11008, "dtype": "bf16", "act": "silu", "residual": True},
        # Prefill: the largest call.
        {"name": "ffn_prefill_8k", "kind": "ffn", "mode": "fwd", "M": 8192, "hidden": 8192, "F": 22016, "dtype": "bf16", "act": "silu", "residual": True},
        # A training step of the 16-head model's block, an odd number of tokens, fp16.
        {"name": "ffn_train_odd", "kind": "ffn", "mode": "train", "M": 8191, "hidden": 1024, "F": 2816, "dtype": "fp16", "act": "silu", "residual": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the listed ranges; work is capped below the largest listed case of its kind."""
    kind = rng.choice(["norm", "rope", "linear", "ffn"])
    if kind == "norm":
        hidden = rng.choice([768, 1024, 4096, 8192]) if rng.random() < 0.7 else _log(rng, 65, 8192)
        mode = rng.choice(["fwd", "fp8", "train"])
        dtype = rng.choice(["bf16", "fp16", "fp32"])
        return {"kind": kind, "mode": mode, "rows": _log(rng, 1, 16384 if mode != "train" else 8192), "hidden": hidden, "dtype": dtype,
                "wdtype": rng.choice([dtype, "fp32"]), "residual": rng.random() < 0.7}
    if kind == "rope":
        H, Hkv, D = rng.choice([(64, 4, 128), (64, 4, 64), (16, 1, 64), (12, 1, 64), (8, 2, 128)])
        axes = rng.choice([1, 2, 3, 3, 4])
        cuts = sorted(rng.sample(range(1, D // 2), axes - 1))
        sections = [b - a for a, b in zip([0] + cuts, cuts + [D // 2])]
        mode = rng.choice(["fwd", "fwd", "train"])
        B = rng.choice([1, 2, 4, 8])
        return {"kind": kind, "mode": mode, "B": B, "T": _log(rng, 1, (16384 if mode == "train" else 32768) // B), "H": H, "Hkv": Hkv, "D": D,
                "sections": ",".join(map(str, sections)), "dtype": rng.choice(["bf16", "fp16", "fp32"]), "far": _log(rng, 1, 1000000)}
    if kind == "linear":
        odd = rng.random() < 0.2
        K = _log(rng, 65, 4096) if odd else rng.choice([768, 896, 1024, 1152, 2048, 4096, 8192])
        N = _log(rng, 65, 4096) if odd else rng.choice([768, 896, 1024, 1152, 2048, 4096, 8192])
        dtype = rng.choice(["bf16", "bf16", "fp16", "e4m3"])
        mode = "fwd" if dtype == "e4m3" else rng.choice(["fwd", "train"])
        return {"kind": kind, "mode": mode, "M": _log(rng, 1, 8192 if mode == "fwd" else 2048), "K": K, "N": N, "dtype": dtype, "bias": rng.random() < 0.5,
                "act": rng.choice(["", "", "silu", "gelu_tanh", "relu"]), "residual": rng.random() < 0.5}
    hidden, F = rng.choice([(768, 2048), (1024, 2816), (2048, 5632), (4096, 11008), (1000, 2730), (8192, 22016)])
    mode = "fwd" if hidden == 8192 else rng.choice(["fwd", "fwd", "train"])
    return {"kind": kind, "mode": mode, "M": _log(rng, 1, 4096), "hidden": hidden, "F": F, "dtype": rng.choice(["bf16", "bf16", "fp16"]),
            "act": rng.choice(["silu", "silu", "gelu_tanh", "relu"]), "residual": rng.random() < 0.6}


# ---------------------------------------------------------------- inputs

def _rows_to_fp8(x):
    s = x.float().abs().amax(-1).clamp_min(1e-12) / E4M3_MAX
    return (x.float() / s[:, None]).to(torch.float8_e4m3fn), s


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed))
    dt = DTYPES[case["dtype"]]
    train = case["mode"] == "train"

    def normal(*shape, std=1.0, dtype=dt):
        return (torch.randn(shape, generator=g, device=dev, dtype=torch.bfloat16 if dtype == torch.bfloat16 else torch.float32) * std).to(dtype)

    s = {"kind": case["kind"], "mode": case["mode"]}
    if case["kind"] == "norm":
        R, N, wdt = case["rows"], case["hidden"], DTYPES[case["wdtype"]]
        s["x"] = normal(R, N)
        # the residual stream: rows of different size, and a few channels that are much larger than the others
        size = torch.exp2(torch.randint(-1, 4, (R, 1), generator=g, device=dev).float())
        channel = 1.0 + 15.0 * (torch.rand((1, N), generator=g, device=dev) < 0.002).float()
        s["res"] = (normal(R, N, dtype=torch.float32) * size * channel).to(dt) if case["residual"] else None
        s["w"] = (1.0 + 0.1 * torch.randn((N,), generator=g, device=dev)).to(wdt)
        if train:
            s["dy"] = normal(R, N)
            s["dh"] = normal(R, N) if case["residual"] else None
        leaves = ("x", "res", "w")
    elif case["kind"] == "rope":
        B, T, H, Hkv, D = (case[k] for k in ("B", "T", "H", "Hkv", "D"))
        s["sections"] = tuple(int(v) for v in case["sections"].split(","))
        packed = normal(B, T, H + 2 * Hkv, D)
        if train:
            s["q"], s["k"], s["v"] = (t.contiguous() for t in packed.split([H, Hkv, Hkv], dim=2))
        else:
            s["q"], s["k"], s["v"] = packed.split([H, Hkv, Hkv], dim=2)
        # patches of 24 x 40 a frame, row by row, behind `far` positions of text (another count for each sequence)
        start = torch.randint(0, case["far"], (B, 1), generator=g, device=dev) + case["far"] // 2
        at = torch.arange(T, device=dev)[None]
        axes = torch.stack([at // 960, at // 40 % 24, at % 40, at % 7])[:len(s["sections"])]
        s["pos"] = (axes + start[None]).contiguous() if len(s["sections"]) > 1 else (at + start)[None].contiguous()
        s["inv_freq"] = BASE ** (-torch.arange(0, D, 2, device=dev, dtype=torch.float64) / D)
        s["dtype"] = torch.float16 if case["dtype"] == "fp16" else torch.bfloat16
        if train:
            s["dq"], s["dk"], s["dv"] = (normal(B, h, T, D, dtype=s["dtype"]) for h in (H, Hkv, Hkv))
        leaves = ("q", "k", "v")
    elif case["kind"] == "linear":
        M, K, N = case["M"], case["K"], case["N"]
        s["act"] = case["act"] or None
        if dt == torch.float8_e4m3fn:
            (s["x"], s["xs"]), (s["w"], s["ws"]) = _rows_to_fp8(normal(M, K, dtype=torch.bfloat16)), _rows_to_fp8(normal(N, K, std=K ** -0.5, dtype=torch.bfloat16))
            dt = torch.bfloat16
        else:
            s["x"], s["w"], s["xs"], s["ws"] = normal(M, K), normal(N, K, std=K ** -0.5), None, None
        s["bias"] = normal(N, std=0.5, dtype=dt) if case["bias"] else None
        s["res"] = normal(M, N, dtype=dt) if case["residual"] else None
        s["dtype"] = dt
        if train:
            s["dy"] = normal(M, N)
        leaves = ("x", "w", "bias", "res")
    else:
        M, N, F = case["M"], case["hidden"], case["F"]
        s["act"] = case["act"]
        s["x"] = normal(M, N)
        s["wg"], s["wu"], s["wd"] = normal(F, N, std=N ** -0.5), normal(F, N, std=N ** -0.5), normal(N, F, std=F ** -0.5)
        s["res"] = normal(M, N) if case["residual"] else None
        if train:
            s["dy"] = normal(M, N)
        leaves = ("x", "wg", "wu", "wd", "res")
    if train:
        s["leaves"] = [s[n].requires_grad_(True) for n in leaves if s[n] is not None]
    return s


# ---------------------------------------------------------------- one pass

def run(s):
    with torch.set_grad_enabled(own and s["mode"] == "train"):
        return {"norm": _norm, "rope": _rope, "linear": _linear, "ffn": _ffn}[s["kind"]](s)


def _act(z, name):
    """(act(z), act'(z))"""
    if name is None:
        return z, None
    if name == "relu":
        return z.clamp_min(0), (z > 0).to(z.dtype)
    if name == "silu":
        p = 1 / (1 + torch.exp(-z))
        return z * p, p * (1 + z * (1 - p))
    c, a = math.sqrt(2 / math.pi), 0.044715
    t = torch.tanh(c * (z + a * z * z * z))
    return 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * a * z * z)


def _norm(s):
    x, res, w = s["x"], s["res"], s["w"]
    if own:
        import nsa_from_scratch_b200 as nsa
        if s["mode"] == "fp8":
            return nsa.rms_norm_fp8(x, w, residual=res, eps=EPS)
        y = nsa.rms_norm(x, w, residual=res, eps=EPS)
        if s["mode"] == "fwd":
            return y
        if res is None:
            return (y.detach(), *torch.autograd.grad(y, s["leaves"], s["dy"]))
        return (y[0].detach(), y[1].detach(), *torch.autograd.grad(y, s["leaves"], (s["dy"], s["dh"])))
    h = x if res is None else (x.float() + res.float()).to(res.dtype)       # the stream as it is stored, which is what is normed
    hf, wf = h.float(), w.float()
    r = torch.rsqrt((hf * hf).mean(-1, keepdim=True) + EPS)
    y = hf * r * wf
    tail = () if res is None else (h,)
    if s["mode"] == "fp8":
        scale = y.abs().amax(-1).clamp_min(1e-12) / E4M3_MAX
        return ((y / scale[:, None]).to(torch.float8_e4m3fn), scale, *tail)
    if s["mode"] == "fwd":
        return y.to(x.dtype) if res is None else (y.to(x.dtype), h)
    dy = s["dy"].float()
    n = hf * r
    u = dy * wf
    dx = r * (u - n * (u * n).mean(-1, keepdim=True))
    dw = (dy * n).sum(0).to(w.dtype)
    if res is None:
        return y.to(x.dtype), dx.to(x.dtype), dw
    dx = dx + s["dh"].float()
    return y.to(x.dtype), h, dx.to(x.dtype), dx.to(res.dtype), dw


def _rope(s):
    q, k, v, pos, inv, sections = s["q"], s["k"], s["v"], s["pos"], s["inv_freq"], s["sections"]
    if own:
        import nsa_from_scratch_b200 as nsa
        out = nsa.rope_axes_to_heads(q, k, v, pos, inv, sections, dtype=s["dtype"])
        if s["mode"] == "fwd":
            return out
        return (*(t.detach() for t in out), *torch.autograd.grad(out, s["leaves"], (s["dq"], s["dk"], s["dv"])))
    axis = torch.repeat_interleave(torch.arange(len(sections), device=q.device), torch.tensor(sections, device=q.device))
    angle = pos.double()[axis].permute(1, 2, 0) * inv                        # [B,T,D/2], radians
    c, sn = angle.cos().float()[:, :, None], angle.sin().float()[:, :, None]

    def turn(x, sn):
        a, b = x.float().chunk(2, dim=-1)
        return torch.cat((a * c - b * sn, b * c + a * sn), dim=-1)

    out = (turn(q, sn), turn(k, sn), v)
    out = tuple(t.to(s["dtype"]).transpose(1, 2).contiguous() for t in out)
    if s["mode"] == "fwd":
        return out
    back = (turn(s["dq"].transpose(1, 2), -sn), turn(s["dk"].transpose(1, 2), -sn), s["dv"].transpose(1, 2))
    return (*out, *(t.to(q.dtype).contiguous() for t in back))


def _linear(s):
    x, w, bias, res = s["x"], s["w"], s["bias"], s["res"]
    if own:
        import nsa_from_scratch_b200 as nsa
        if s["xs"] is not None:
            return nsa.linear_fp8(x, w, s["xs"], s["ws"], bias, activation=s["act"], residual=res, dtype=s["dtype"])
        y = nsa.linear(x, w, bias, activation=s["act"], residual=res)
        return y if s["mode"] == "fwd" else (y.detach(), *torch.autograd.grad(y, s["leaves"], s["dy"]))
    xf, wf = x.float(), w.float()
    z = xf @ wf.T
    if s["xs"] is not None:
        z = z * s["xs"][:, None] * s["ws"]
    if bias is not None:
        z = z + bias.float()
    y, slope = _act(z, s["act"])
    if res is not None:
        y = y + res.float()
    y = y.to(s["dtype"])
    if s["mode"] == "fwd":
        return y
    dz = s["dy"].float()
    if slope is not None:
        dz = dz * slope
    grads = [(dz @ wf).to(x.dtype), (dz.T @ xf).to(w.dtype)]
    if bias is not None:
        grads.append(dz.sum(0).to(bias.dtype))
    if res is not None:
        grads.append(s["dy"].to(res.dtype))
    return (y, *grads)


def _ffn(s):
    x, wg, wu, wd, res = s["x"], s["wg"], s["wu"], s["wd"], s["res"]
    if own:
        import nsa_from_scratch_b200 as nsa
        y = nsa.gated_mlp(x, wg, wu, wd, activation=s["act"], residual=res)
        return y if s["mode"] == "fwd" else (y.detach(), *torch.autograd.grad(y, s["leaves"], s["dy"]))
    xf, gf, uf, df = x.float(), wg.float(), wu.float(), wd.float()
    u = xf @ uf.T
    a, slope = _act(xf @ gf.T, s["act"])
    h = a * u
    y = h @ df.T
    if res is not None:
        y = y + res.float()
    y = y.to(x.dtype)
    if s["mode"] == "fwd":
        return y
    dy = s["dy"].float()
    dh = dy @ df
    dg, du = dh * u * slope, dh * a
    grads = [dg @ gf + du @ uf, dg.T @ xf, du.T @ xf, dy.T @ h]
    if res is not None:
        grads.append(dy)
    return (y, *(t.to(x.dtype) for t in grads))


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    c, train = case, case["mode"] == "train"
    size = {"bf16": 2, "fp16": 2, "fp32": 4, "e4m3": 1}
    isz = size[c["dtype"]]
    if c["kind"] == "norm":
        n = c["rows"] * c["hidden"]
        nbytes = n * isz * (3 if c["residual"] else 1) + n * (1 if c["mode"] == "fp8" else isz) + c["hidden"] * size[c["wdtype"]]
        nbytes += c["rows"] * 4 if c["mode"] == "fp8" else 0
        if train:       # dy (and the stream's gradient) read, one gradient for x and the residual alike, dw
            nbytes += n * isz * (3 if c["residual"] else 2) + c["hidden"] * size[c["wdtype"]]
        return {"bytes": float(nbytes), "flops": float(n * (15 if train else 5))}
    if c["kind"] == "rope":
        n = c["B"] * c["T"] * (c["H"] + 2 * c["Hkv"]) * c["D"]
        axes = len(c["sections"].split(","))
        nbytes = n * (isz + 2) * (2 if train else 1) + axes * c["B"] * c["T"] * 8
        return {"bytes": float(nbytes), "flops": float(3 * n * (2 if train else 1))}
    if c["kind"] == "linear":
        M, K, N = c["M"], c["K"], c["N"]
        nbytes = (M * K + N * K) * isz + M * N * 2 * (2 if c["residual"] else 1) + (N * 2 if c["bias"] else 0)
        nbytes += 4 * (M + N) if c["dtype"] == "e4m3" else 0
        if train:
            nbytes += M * N * 2 * (2 if c["residual"] else 1) + (M * K + N * K) * 2 + (N * 2 if c["bias"] else 0)
        return {"bytes": float(nbytes), "flops": 2.0 * M * K * N * (3 if train else 1)}
    M, N, F = c["M"], c["hidden"], c["F"]
    nbytes = 2 * (M * N * (3 if c["residual"] else 2) + 3 * N * F)
    if train:
        nbytes += 2 * (M * N * (3 if c["residual"] else 2) + 3 * N * F)
    return {"bytes": float(nbytes), "flops": 6.0 * M * N * F * (3 if train else 1)}


# ---------------------------------------------------------------- the definitions in 64 bits

def _act64(z, name):
    if not name:
        return z
    if name == "relu":
        return torch.relu(z)
    return z * torch.sigmoid(z) if name == "silu" else torch.nn.functional.gelu(z, approximate="tanh")


def exact(case, seed):
    s = prepare(case, seed)
    train = s["mode"] == "train"
    d = {k: t.detach().double().requires_grad_(train) if isinstance(t, torch.Tensor) and t.is_floating_point() else t for k, t in s.items()}
    with torch.set_grad_enabled(train):
        if s["kind"] == "norm":
            x, w, h = d["x"], d["w"], d["x"]
            if s["res"] is not None:
                total = d["x"] + d["res"]
                h = total + (total.detach().to(s["res"].dtype).double() - total.detach())      # stored in the stream's type
            y = w * h / (h.square().mean(-1, keepdim=True) + EPS).sqrt()
            if s["mode"] == "fp8":
                scale = y.abs().amax(-1).clamp_min(1e-12) / E4M3_MAX
                return (y / scale[:, None], scale) + (() if s["res"] is None else (h,))
            outs = [y] if s["res"] is None else [y, h]
            wrt, seeds = ([d["x"], w], [d["dy"] if train else None]) if s["res"] is None else ([d["x"], d["res"], w], [d["dy"], d["dh"]] if train else None)
        elif s["kind"] == "rope":
            half, angles, at = case["D"] // 2, [], 0
            for a, n in enumerate(s["sections"]):
                angles.append(s["pos"][a].double()[:, :, None] * s["inv_freq"][at:at + n])
                at += n
            turned = torch.polar(torch.ones((), dtype=torch.float64, device=s["q"].device), torch.cat(angles, -1))[:, None]

            def rotate(x):
                z = torch.complex(x[..., :half], x[..., half:]).transpose(1, 2) * turned
                return torch.cat((z.real, z.imag), -1)

            outs = [rotate(d["q"]), rotate(d["k"]), d["v"].transpose(1, 2)]
            wrt, seeds = [d["q"], d["k"], d["v"]], [d["dq"], d["dk"], d["dv"]] if train else None
        elif s["kind"] == "linear":
            x, w = d["x"], d["w"]
            if s["xs"] is not None:
                x, w = x * d["xs"][:, None], w * d["ws"][:, None]
            y = _act64(torch.nn.functional.linear(x, w, d["bias"]), s["act"])
            outs = [y if s["res"] is None else y + d["res"]]
            wrt, seeds = [d[k] for k in ("x", "w", "bias", "res") if s[k] is not None], [d["dy"]] if train else None
        else:
            lin = torch.nn.functional.linear
            y = lin(_act64(lin(d["x"], d["wg"]), s["act"]) * lin(d["x"], d["wu"]), d["wd"])
            outs = [y if s["res"] is None else y + d["res"]]
            wrt, seeds = [d[k] for k in ("x", "wg", "wu", "wd", "res") if s[k] is not None], [d["dy"]] if train else None
        if train:
            return tuple(t.detach() for t in outs) + torch.autograd.grad(outs, wrt, [t.detach() for t in seeds])
        return outs[0] if len(outs) == 1 else tuple(outs)
