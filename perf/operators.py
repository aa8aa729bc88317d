"""What the training-side operators of the transformer blocks and the text tower are measured on: the token embedding and its
gradient, the norms around a transformer block fused with its gate and residual, and the global gradient norm with clipping.

``own`` selects the side: False = the plain forms below (elementary torch operations in 32 bits, rounded once at the end),
True = the framework's operators (geodiffuser_amd.ops)."""
import math

import torch

own = False

DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
SIZE = {"f16": 2, "bf16": 2, "f32": 4}
EPS = 1e-5


# ---------------------------------------------------------------------------------------------------- the cases
def _embed(name, grad, B, L, V, C, dtype, pos, scale=1.0):
    return dict(name=name, op="embed_grad" if grad else "embed", B=B, L=L, V=V, C=C, dtype=dtype, pos=pos, scale=scale)


def _norm(name, train, B, N, C, dtype, kind, gate, post, res_scale=1.0):
    return dict(name=name, op="norm_train" if train else "norm", B=B, N=N, C=C, dtype=dtype, kind=kind, gate=gate, post=post, res_scale=res_scale)


def _clip(name, width, layers, V, dtype, vectors, max_norm):
    return dict(name=name, op="clip", width=width, layers=layers, V=V, dtype=dtype, vectors=vectors, max_norm=max_norm)


def listed():
    return [
        # one prompt through the SD2.1 text tower's embedding (every edit's first step): latency
        _embed("embed-prompt", False, 1, 77, 49408, 1024, "bf16", True),
        # a large batch of prompts at the width of SDXL's second tower: bandwidth
        _embed("embed-batch", False, 1024, 77, 49408, 1280, "f16", True),
        # four prompts' gradient into the whole f32 table of an SD1-width tower (learning a token): zero rows and latency
        _embed("embed-grad-prompts", True, 4, 77, 49408, 768, "f32", False),
        # a training batch whose prompts are mostly padding: one token with half of all rows, and the position gradient
        _embed("embed-grad-batch", True, 2048, 77, 49408, 1024, "bf16", True),
        # residual add and next norm of one prompt in the text tower: latency
        _norm("norm-prompt", False, 1, 77, 1024, "bf16", "layer", "none", False),
        # the 64 x 64 level of the UNet with a per-sample gate and a norm on the block's output
        _norm("norm-gated", False, 2, 4096, 320, "f16", "layer", "sample", True),
        # training pass at the 32 x 32 level with a per-channel gate (layer scale)
        _norm("norm-train", True, 4, 1024, 640, "bf16", "layer", "channel", False),
        # training at SDXL's width in 32 bits, RMS norms on both sides of the block
        _norm("norm-train-wide", True, 8, 4096, 1280, "f32", "rms", "sample", True, 0.70710678),
        # odd sizes: no row is a whole number of vectors
        _norm("norm-train-ragged", True, 3, 257, 333, "f16", "rms", "sample", False),
        # the null-text optimisation's one [1, 77, 1024] embedding: latency
        _clip("clip-embedding", 1024, 0, 77, "f32", False, 0.1),
        # every gradient of SD2.1's text tower: 16-bit matrices, 32-bit vectors
        _clip("clip-text-tower", 1024, 23, 49408, "bf16", True, 1.0),
        # every gradient of SDXL's second text tower
        _clip("clip-wide-tower", 1280, 32, 49408, "bf16", False, 1.0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """A channel count: a multiple of 64 as the models have them, or any."""
    c = _log(rng, lo, hi)
    return max(lo, c // 64 * 64) if rng.random() < 0.6 else c


def draw(rng):
    dtype = rng.choice(["f16", "bf16", "f32"])
    what = rng.random()
    if what < 0.35:
        B, L, C = _log(rng, 1, 2048), rng.randint(1, 77), _width(rng, 32, 1280)
        B = max(1, min(B, 200_000_000 // (L * C)))
        c = _embed("", rng.random() < 0.6, B, L, _log(rng, 1000, 49408), C, dtype, rng.random() < 0.5, rng.choice([1.0, 8.0, C ** 0.5]))
    elif what < 0.75:
        B, N, C = rng.randint(1, 8), _log(rng, 1, 4096), _width(rng, 32, 2048)
        N = max(1, min(N, 40_000_000 // (B * C)))
        c = _norm("", rng.random() < 0.6, B, N, C, dtype, rng.choice(["layer", "rms"]), rng.choice(["none", "channel", "sample"]),
                  rng.random() < 0.5, rng.choice([1.0, 0.70710678, 2.0]))
    else:
        w = _width(rng, 48, 1280)
        layers = rng.randint(0, min(24, 250_000_000 // (12 * w * w)))
        c = _clip("", w, layers, _log(rng, 77, 49408), dtype, rng.random() < 0.5, rng.choice([0.1, 1.0, 1e4]))
    del c["name"]
    return c


def _tower(case):
    """The parameter shapes of a text tower: embedding, positions, then 12 tensors a layer and the final norm."""
    w = case["width"]
    shapes = [(case["V"], w)]
    if case["layers"]:
        shapes += [(77, w)] + [(3 * w, w), (3 * w,), (w, w), (w,), (w,), (w,), (w,), (w,), (4 * w, w), (4 * w,), (w, 4 * w), (w,)] * case["layers"] + [(w,), (w,)]
    return shapes


# ---------------------------------------------------------------------------------------------------- inputs
def _make(case, seed, device):
    g = torch.Generator(device=device).manual_seed(seed)

    def normal(*shape, std=1.0, mean=0.0, dtype=None):
        return (torch.randn(*shape, generator=g, device=device) * std + mean).to(dtype or dt)

    s = {"case": case}
    dt = DT[case["dtype"]]
    if case["op"] in ("embed", "embed_grad"):
        B, L, V, C = (case[k] for k in "BLVC")
        # prompts as a tokenizer lays them out: a begin token, words (frequent ones small), an end token, padding 0 behind it
        u = torch.rand(B, L, generator=g, device=device)
        ids = (2 + (V - 4) * u ** 4).long().clamp(max=V - 3)
        n = torch.randint(1, max(2, L), (B, 1), generator=g, device=device)
        at = torch.arange(L, device=device)
        ids = torch.where(at == 0, V - 2, torch.where(at < n, ids, torch.where(at == n, V - 1, 0)))
        s["ids"] = ids.contiguous()
        if case["op"] == "embed":
            s["table"] = normal(V, C, std=0.02)
            s["pos"] = normal(77, C, std=0.01) if case["pos"] else None
        else:
            s["dy"] = normal(B, L, C, std=1e-2)
    elif case["op"] in ("norm", "norm_train"):
        B, N, C = (case[k] for k in "BNC")
        s["x"], s["res"] = normal(B, N, C, std=0.7, mean=0.1), normal(B, N, C, std=1.5)
        s["gate"] = None if case["gate"] == "none" else normal(C, std=0.3, mean=0.8) if case["gate"] == "channel" else normal(B, C, std=0.3, mean=0.8)
        layer = case["kind"] == "layer"
        for k in ("pre", "post"):
            there = k == "pre" or case["post"]
            s[k + "_gamma"] = normal(C, std=0.2, mean=1.0) if there else None
            s[k + "_beta"] = normal(C, std=0.1) if there and layer else None
        if case["op"] == "norm_train":
            s["gy"], s["gs"] = normal(B, N, C), normal(B, N, C, std=0.5)
    else:
        # gradients as views of one buffer for each type, 16-byte aligned, and the buffers that the optimiser reads
        shapes = _tower(case)
        types = [torch.float32 if case["vectors"] and len(sh) == 1 else dt for sh in shapes]
        s["grads"], s["outs"], s["flat"] = [None] * len(shapes), [None] * len(shapes), []
        for t in sorted(set(types), key=str):
            at, total = {}, 0
            for i, sh in enumerate(shapes):
                if types[i] == t:
                    at[i] = total
                    total += -(-math.prod(sh) // 16) * 16
            flat, out = torch.zeros(total, dtype=t, device=device), torch.zeros(total, dtype=t, device=device)
            for i, o in at.items():
                n = math.prod(shapes[i])
                s["grads"][i], s["outs"][i] = flat[o:o + n].view(shapes[i]), out[o:o + n].view(shapes[i])
                s["grads"][i].normal_(0, 1e-3 if len(shapes[i]) > 1 else 1e-2, generator=g)
            s["flat"].append(out)
    return s


def prepare(case, seed):
    return _make(case, seed, "cuda")


# ---------------------------------------------------------------------------------------------------- plain forms
def _plain_norm(v, kind, gamma, beta):
    """-> (output, normalised rows, 1 / deviation) in 32 bits."""
    if kind == "layer":
        v = v - v.mean(-1, keepdim=True)
    r = torch.rsqrt((v * v).mean(-1, keepdim=True) + EPS)
    xh = v * r
    y = xh * gamma.float()
    return (y if beta is None else y + beta.float()), xh, r


def _plain_norm_grad(g, gamma, xh, r, kind):
    g = g * gamma.float()
    d = g - xh * (g * xh).mean(-1, keepdim=True)
    return r * (d - g.mean(-1, keepdim=True) if kind == "layer" else d)


def _plain(s):
    case = s["case"]
    dt = DT[case["dtype"]]
    if case["op"] == "embed":
        y = s["table"][s["ids"]].float() * case["scale"]
        return (y if s["pos"] is None else y + s["pos"][:case["L"]].float()).to(dt)
    if case["op"] == "embed_grad":
        # a 32-bit running sum over tens of thousands of rows (padding) is further off than a 32-bit result may be
        acc = torch.float64 if case["dtype"] == "f32" and case["B"] * case["L"] > 4096 else torch.float32
        dy = s["dy"].to(acc)
        d = torch.zeros(case["V"], case["C"], dtype=acc, device=dy.device)
        d.index_add_(0, s["ids"].reshape(-1), dy.reshape(-1, case["C"]))
        out = [(d * case["scale"]).to(dt)]
        if case["pos"]:
            p = torch.zeros(77, case["C"], dtype=dt, device=dy.device)
            p[:case["L"]] = dy.sum(0).to(dt)
            out.append(p)
        return out
    if case["op"] == "clip":
        total = torch.stack([t.float().square().sum() for t in s["grads"]]).sum().sqrt()
        factor = (case["max_norm"] / (total + 1e-6)).clamp(max=1.0)
        for t, o in zip(s["grads"], s["outs"]):
            o.copy_(t.float() * factor)
        return [total] + s["flat"]
    kind, x = case["kind"], s["x"].float()
    gate = None if s["gate"] is None else s["gate"].float() if case["gate"] == "channel" else s["gate"].float()[:, None]
    h, xh, xr = _plain_norm(x, kind, s["post_gamma"], s["post_beta"]) if case["post"] else (x, None, None)
    st = case["res_scale"] * s["res"].float() + (h if gate is None else gate * h)
    y, sh, sr = _plain_norm(st, kind, s["pre_gamma"], s["pre_beta"])
    out = {"s": st.to(dt), "y": y.to(dt)}
    if case["op"] == "norm":
        return out
    gy = s["gy"].float()
    ds = _plain_norm_grad(gy, s["pre_gamma"], sh, sr, kind) + s["gs"].float()
    out["dpre_gamma"] = (gy * sh).sum((0, 1)).to(dt)
    if s["pre_beta"] is not None:
        out["dpre_beta"] = gy.sum((0, 1)).to(dt)
    out["dres"] = (case["res_scale"] * ds).to(dt)
    dh = ds
    if gate is not None:
        out["dgate"] = (ds * h).sum((0, 1) if case["gate"] == "channel" else 1).to(dt)
        dh = gate * ds
    if case["post"]:
        out["dpost_gamma"] = (dh * xh).sum((0, 1)).to(dt)
        if s["post_beta"] is not None:
            out["dpost_beta"] = dh.sum((0, 1)).to(dt)
        dh = _plain_norm_grad(dh, s["post_gamma"], xh, xr, kind)
    out["dx"] = dh.to(dt)
    return out


# ---------------------------------------------------------------------------------------------------- the framework's operators
def _own(s):
    from geodiffuser_amd import ops
    case = s["case"]
    if case["op"] == "embed":
        return ops.embed_tokens(s["ids"], s["table"], s["pos"], scale=case["scale"])
    if case["op"] == "embed_grad":
        out = [ops.embed_tokens_bwd(s["ids"], s["dy"], case["V"], scale=case["scale"])]
        if case["pos"]:
            out.append(ops.embed_positions_bwd(s["dy"], 77))
        return out
    if case["op"] == "clip":
        return [ops.clip_grad_norm(s["grads"], case["max_norm"], out=s["outs"])] + s["flat"]
    pre = ops.Norm(case["kind"], s["pre_gamma"], s["pre_beta"], EPS)
    post = ops.Norm(case["kind"], s["post_gamma"], s["post_beta"], EPS) if case["post"] else None
    st, y, stats = ops.block_norm(s["x"], s["res"], pre, post=post, gate=s["gate"], res_scale=case["res_scale"])
    out = {"s": st, "y": y}
    if case["op"] == "norm_train":
        d = ops.block_norm_bwd(s["x"], s["res"], s["gy"], s["gs"], stats, pre, post=post, gate=s["gate"], res_scale=case["res_scale"])
        out.update({k: v for k, v in d.items() if v is not None})
    return out


def run(state):
    return _own(state) if own else _plain(state)


# ---------------------------------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    z = SIZE[case["dtype"]]
    if case["op"] in ("embed", "embed_grad"):
        n, L, V, C = case["B"] * case["L"], case["L"], case["V"], case["C"]
        if case["op"] == "embed":
            return {"bytes": 8 * n + (min(n, V) + n + (L if case["pos"] else 0)) * C * z, "flops": 2 * n * C}
        return {"bytes": 8 * n + (n + V + (77 if case["pos"] else 0)) * C * z, "flops": (2 if case["pos"] else 1) * n * C}
    if case["op"] == "clip":
        n = n16 = 0
        for sh in _tower(case):
            k = math.prod(sh)
            n, n16 = n + k, n16 + k * (4 if case["vectors"] and len(sh) == 1 else z)
        return {"bytes": 2 * n16, "flops": 3 * n}
    n = case["B"] * case["N"] * case["C"]
    # forward: x, res in, s, y out; training besides: gy, gs in, dx, dres out and x, res a second time
    return {"bytes": (10 if case["op"] == "norm_train" else 4) * n * z, "flops": (40 if case["op"] == "norm_train" else 14) * n}


# ---------------------------------------------------------------------------------------------------- the definition in 64 bits
def exact(case, seed):
    s = {k: v.double() if torch.is_tensor(v) and v.is_floating_point() else v for k, v in _make(case, seed, "cuda").items()}
    if case["op"] == "embed":
        rows = torch.index_select(s["table"], 0, s["ids"].flatten()).reshape(case["B"], case["L"], case["C"])
        return torch.add(0 if s["pos"] is None else s["pos"][None, :case["L"]], rows, alpha=case["scale"])
    if case["op"] == "embed_grad":
        order = torch.sort(s["ids"].flatten(), stable=True)
        count = torch.bincount(order.values, minlength=case["V"])
        rows = s["dy"].reshape(-1, case["C"])[order.indices]
        d = torch.segment_reduce(rows, "sum", lengths=count, axis=0, initial=0.0) * case["scale"]
        if not case["pos"]:
            return [d]
        return [d, torch.cat([s["dy"].sum(0), s["dy"].new_zeros(77 - case["L"], case["C"])])]
    if case["op"] == "clip":
        total = math.sqrt(sum(float(torch.linalg.vector_norm(t, dtype=torch.float64)) ** 2 for t in s["grads"]))
        factor = min(1.0, case["max_norm"] / (total + 1e-6))
        for t, o in zip(s["grads"], s["outs"]):
            o.copy_(t)
        return [torch.tensor(total, dtype=torch.float64)] + [f.double() * factor for f in s["flat"]]

    def norm(v, gamma, beta):
        if case["kind"] == "layer":
            return torch.nn.functional.layer_norm(v, v.shape[-1:], gamma, beta, EPS)
        return v / (v.pow(2).mean(-1, keepdim=True) + EPS).sqrt() * gamma

    leaf = {k: v.requires_grad_() for k, v in s.items() if torch.is_tensor(v) and k not in ("gy", "gs")}
    h = norm(leaf["x"], leaf["post_gamma"], leaf.get("post_beta")) if case["post"] else leaf["x"]
    if "gate" in leaf:
        h = h * (leaf["gate"] if case["gate"] == "channel" else leaf["gate"].unsqueeze(1))
    st = leaf["res"] * case["res_scale"] + h
    y = norm(st, leaf["pre_gamma"], leaf.get("pre_beta"))
    out = {"s": st.detach(), "y": y.detach()}
    if case["op"] == "norm_train":
        names = list(leaf)
        for k, d in zip(names, torch.autograd.grad([st, y], [leaf[k] for k in names], [s["gs"], s["gy"]])):
            out["d" + k] = d
    return out
