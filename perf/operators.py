"""The operators around and inside a mixture-of-experts layer, as they are measured.

Three operators, by a case's "op":

  block_norm      norms behind and before a block, fused with its gate and residual scale
                  ("block_norm_backward": its gradients)
  grouped_mm      one product per expert over ragged row segments ("grouped_mm_dgrad" and
                  "grouped_mm_wgrad": its two gradients)
  expert_linear_w4  products with 4-bit weights and group scales for few tokens, each slot with
                  its own expert

`own` false: the plain form in torch, 32 bits; true: the calls of moe_b200.
"""
import math
import os
import sys

import torch

own = False

EPS = 1e-6


def _mb():
    if "moe_b200" not in sys.modules:
        root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "15618-final_b200")
        if root not in sys.path:
            sys.path.insert(0, root)
    import moe_b200
    return moe_b200


# ------------------------------------------------------------------ cases ----

def listed():
    norm = dict(op="block_norm", post=True, pre=True, gate="none", residual="bfloat16", scale=1.0)
    mm = dict(K=4, E=60, dist="zipf", dtype="bfloat16")
    return [
        # one decode step of a batch of 16: the launch is the cost
        dict(norm, name="norm_decode", T=16, d=2048, dtype="bfloat16"),
        # the prompt batch of the full-layer workload (16384 tokens of 2048), a gate per token
        dict(norm, name="norm_prompt", T=16384, d=2048, dtype="bfloat16", gate="token", scale=0.5),
        # training: 8192 tokens of 4096, a learned gate per channel
        dict(norm, name="norm_backward", op="block_norm_backward", T=8192, d=4096, dtype="bfloat16", gate="channel", scale=0.7),
        # a short odd batch with an odd width and a 32-bit residual stream
        dict(norm, name="norm_backward_odd", op="block_norm_backward", T=777, d=1001, dtype="float16", gate="full",
             residual="float32", scale=1.25),
        # a decode batch of 32 tokens through 16-bit experts: two rows an expert, the weights' bytes are the cost
        dict(mm, name="mm_few_rows", op="grouped_mm", T=32, d=2048, N=2816),
        # the gate/up product of the full-layer workload
        dict(mm, name="mm_prompt", op="grouped_mm", T=16384, d=2048, N=2816),
        # its gradients in training: the gate/up product's input, and its weights
        dict(mm, name="mm_dgrad", op="grouped_mm_dgrad", T=16384, d=2048, N=2816),
        dict(mm, name="mm_wgrad", op="grouped_mm_wgrad", T=16384, d=2048, N=2816),
        # many experts with short ragged segments (some of them empty), sizes in no power of two
        dict(op="grouped_mm_wgrad", name="mm_wgrad_ragged", T=999, K=8, E=128, dist="zipf", dtype="float16", d=1096, N=712),
        # a single token: gate/up product with its SwiGLU, four experts read
        dict(op="expert_linear_w4", name="w4_token", T=1, K=4, E=60, dist="zipf", d=2048, N=2816, group=128, act="swiglu",
             zeros=False, per_slot=False, dtype="bfloat16"),
        # a decode batch of 64: nearly every expert read
        dict(op="expert_linear_w4", name="w4_batch", T=64, K=4, E=60, dist="uniform", d=2048, N=2816, group=128, act="swiglu",
             zeros=False, per_slot=False, dtype="bfloat16"),
        # the down product of an odd batch with small groups and zero points, one input row for each slot
        dict(op="expert_linear_w4", name="w4_down", T=147, K=4, E=60, dist="zipf", d=1408, N=2048, group=32, act="none",
             zeros=True, per_slot=True, dtype="float16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["block_norm", "block_norm_backward", "grouped_mm", "grouped_mm_dgrad", "grouped_mm_wgrad", "expert_linear_w4",
                     "expert_linear_w4"])
    dtype = rng.choice(["bfloat16", "float16"])
    if op.startswith("block_norm"):
        d = _log(rng, 64, 8192)
        if rng.random() < 0.7:
            d = max(8, d // 8 * 8)
        T = min(_log(rng, 1, 32768), 8192 * 4096 // d)
        post = rng.random() < 0.7
        return dict(op=op, T=T, d=d, dtype=dtype, post=post, pre=rng.random() < 0.8 or not post,
                    gate=rng.choice(["none", "token", "channel", "full"]), residual=rng.choice([dtype, "float32"]),
                    scale=round(rng.uniform(0.2, 1.5), 3))
    if op.startswith("grouped_mm"):
        d, N = (max(1, _log(rng, 64, 4096) // 8) * 8 for _ in range(2))
        E = min(_log(rng, 1, 128), 60 * 2048 * 2816 // (d * N))
        K = rng.randint(1, min(8, E))
        T = _log(rng, 1, 16384)
        T = max(1, min(T, 16384 * 4 * 2048 * 2816 // (K * d * N)))
        return dict(op=op, T=T, K=K, E=E, d=d, N=N, dist=rng.choice(["zipf", "uniform"]), dtype=dtype)
    group = rng.choice([32, 64, 128])
    d = max(1, _log(rng, 128, 4096) // group) * group
    act = rng.choice(["swiglu", "none"])
    N = max(1, _log(rng, 64, 4096) // 16) * 16
    E = min(_log(rng, 4, 128), 60 * 2048 * 2816 // (d * N))
    K = rng.randint(1, min(8, E))
    return dict(op=op, T=max(1, min(_log(rng, 1, 192), 600 // K)), K=K, E=E, d=d, N=N, group=group, act=act,
                zeros=rng.random() < 0.5, per_slot=rng.random() < 0.5, dist=rng.choice(["zipf", "uniform"]), dtype=dtype)


# ----------------------------------------------------------------- inputs ----

def _routing(c, g):
    """Experts [T, K] of each token, the most likely first (Gumbel top-K; expert popularity 1/rank^1.2 or even)."""
    u = torch.rand((c["T"], c["E"]), generator=g, device="cuda", dtype=torch.float64).clamp_min_(1e-12)
    score = -torch.log(-torch.log(u))
    if c["dist"] == "zipf":
        score -= 1.2 * torch.log(torch.arange(1, c["E"] + 1, device="cuda", dtype=torch.float64))
    return score.topk(c["K"], dim=1).indices.to(torch.int32).contiguous()


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    dt = getattr(torch, c["dtype"])

    def rand(shape, scale=1.0, to=dt, at=0.0):
        return (torch.randn(shape, generator=g, device="cuda") * scale + at).to(to)

    s = dict(c)
    if c["op"].startswith("block_norm"):
        T, d, res = c["T"], c["d"], getattr(torch, c["residual"])
        s["residual"] = rand((T, d), 1.5, res)
        s["y"] = rand((T, d), 0.7)
        s["w_post"] = rand((d,), 0.2, at=1.0) if c["post"] else None
        s["w_pre"] = rand((d,), 0.2, at=1.0) if c["pre"] else None
        shape = {"none": None, "token": (T, 1), "channel": (1, d), "full": (T, d)}[c["gate"]]
        s["gate"] = None if shape is None else rand(shape, 0.3, at=0.6)
        if c["op"] == "block_norm_backward":
            s["residual_out"] = s.pop("residual")
            s["d_residual_out"] = rand((T, d), 0.1, res)
            s["d_normed"] = rand((T, d), 0.1) if c["pre"] else None
        return s
    if c["op"].startswith("grouped_mm"):
        rows, d, N, E = c["T"] * c["K"], c["d"], c["N"], c["E"]
        counts = torch.bincount(_routing(c, g).flatten(), minlength=E)
        s["seg_start"] = torch.cat([counts.new_zeros(1), counts.cumsum(0)]).to(torch.int32)
        s["sizes"] = counts.tolist()
        if c["op"] != "grouped_mm_dgrad":
            s["x"] = rand((rows, d))
        if c["op"] != "grouped_mm":
            s["dy"] = rand((rows, N))
        if c["op"] != "grouped_mm_wgrad":
            s["w"] = rand((E, N, d), 0.02)
        return s
    T, K, E, d, N, G = (c[k] for k in ("T", "K", "E", "d", "N", "group"))
    s["asgn"] = _routing(c, g)
    s["x"] = rand((T, K, d) if c["per_slot"] else (T, d))
    s["w_q"] = torch.randint(0, 256, (E, N, d // 2), generator=g, device="cuda", dtype=torch.uint8)
    s["w_scale"] = ((0.5 + torch.rand((E, N, d // G), generator=g, device="cuda")) * 0.006).to(dt)
    s["w_zero"] = torch.randint(0, 16, (E, N, d // G), generator=g, device="cuda", dtype=torch.uint8) if c["zeros"] else None
    return s


# -------------------------------------------------------------------- run ----

def run(s):
    return _own(s) if own else _PLAIN[s["op"]](s)


def _own(s):
    mb = _mb()
    op = s["op"]
    if op == "block_norm":
        r = mb.block_norm(s["residual"], s["y"], w_post=s["w_post"], w_pre=s["w_pre"], gate=s["gate"], scale=s["scale"], eps=EPS)
        return {"residual_out": r.residual_out, "normed": r.normed}
    if op == "block_norm_backward":
        r = mb.block_norm_backward(s["d_residual_out"], s["d_normed"], s["residual_out"], s["y"], w_post=s["w_post"],
                                   w_pre=s["w_pre"], gate=s["gate"], scale=s["scale"], eps=EPS)
        return {"d_residual": r.d_residual, "d_y": r.d_y, "d_w_post": r.d_w_post, "d_w_pre": r.d_w_pre, "d_gate": r.d_gate}
    if op == "grouped_mm":
        return mb.grouped_mm(s["x"], s["seg_start"], s["w"])
    if op == "grouped_mm_dgrad":
        return mb.grouped_mm_dgrad(s["dy"], s["seg_start"], s["w"])
    if op == "grouped_mm_wgrad":
        return mb.grouped_mm_wgrad(s["dy"], s["x"], s["seg_start"])
    return mb.expert_linear_w4(s["x"], s["asgn"], s["w_q"], s["w_scale"], w_zero=s["w_zero"],
                               act="swiglu" if s["act"] == "swiglu" else None)


def _rms(v):
    return torch.rsqrt(v.square().mean(1, keepdim=True) + EPS)


def _plain_block_norm(s):
    z = s["y"].float()
    if s["w_post"] is not None:
        z = z * _rms(z) * s["w_post"].float()
    if s["gate"] is not None:
        z = z * s["gate"].float()
    r = s["residual"].float() + s["scale"] * z
    n = (r * _rms(r) * s["w_pre"].float()).to(s["y"].dtype) if s["w_pre"] is not None else None
    return {"residual_out": r.to(s["residual"].dtype), "normed": n}


def _plain_block_norm_backward(s):
    dt, ds, y = s["y"].dtype, s["d_residual_out"].float(), s["y"].float()
    d_w_pre = d_w_post = d_gate = None
    if s["w_pre"] is not None:
        r, dn = s["residual_out"].float(), s["d_normed"].float()
        c = _rms(r)
        r = r * c
        u = dn * s["w_pre"].float()
        ds = ds + c * (u - r * (u * r).mean(1, keepdim=True))
        d_w_pre = (dn * r).sum(0)
    dz = s["scale"] * ds
    a = _rms(y) if s["w_post"] is not None else None
    yh = y * a if a is not None else y
    if s["gate"] is not None:
        z = yh * s["w_post"].float() if a is not None else y
        d_gate = dz * z
        axis = {(y.shape[0], 1): 1, (1, y.shape[1]): 0}.get(tuple(s["gate"].shape))
        d_gate = d_gate.to(dt) if axis is None else d_gate.sum(axis, keepdim=True)
        dz = dz * s["gate"].float()
    if a is not None:
        d_w_post = (dz * yh).sum(0)
        v = dz * s["w_post"].float()
        dz = a * (v - yh * (v * yh).mean(1, keepdim=True))
    return {"d_residual": ds.to(s["d_residual_out"].dtype), "d_y": dz.to(dt), "d_w_post": d_w_post, "d_w_pre": d_w_pre, "d_gate": d_gate}


def _plain_grouped_mm(s):
    w = s["w"].float()
    return torch.cat([x @ w[e].T for e, x in enumerate(s["x"].float().split(s["sizes"]))]).to(s["x"].dtype)


def _plain_grouped_mm_dgrad(s):
    w = s["w"].float()
    return torch.cat([dy @ w[e] for e, dy in enumerate(s["dy"].float().split(s["sizes"]))]).to(s["dy"].dtype)


def _plain_grouped_mm_wgrad(s):
    dy, x = s["dy"].float().split(s["sizes"]), s["x"].float().split(s["sizes"])
    return torch.stack([a.T @ b for a, b in zip(dy, x)]).to(s["x"].dtype)


def _plain_expert_linear_w4(s):
    T, K, E, G, d = s["T"], s["K"], s["E"], s["group"], s["d"]
    e = s["asgn"].flatten().long()
    few = T * K <= E  # few slots: the weights of each slot; else every expert's product with every row
    pick = (lambda t: t[e]) if few else (lambda t: t)
    q = pick(s["w_q"])
    w = torch.stack([q & 15, q >> 4], dim=-1).flatten(-2).float().unflatten(-1, (d // G, G))
    zero = pick(s["w_zero"]).float().unsqueeze(-1) if s["w_zero"] is not None else 8.0
    w = ((w - zero) * pick(s["w_scale"]).float().unsqueeze(-1)).flatten(-2)
    x = s["x"].float()
    rows = x.reshape(-1, d) if s["per_slot"] else x.repeat_interleave(K, 0)
    if few:
        y = (w @ rows.unsqueeze(-1)).squeeze(-1)
    else:
        y = (rows @ w.transpose(1, 2))[e, torch.arange(T * K, device=e.device)]
    if s["act"] == "swiglu":
        g, u = y.chunk(2, dim=1)
        y = g / (1.0 + torch.exp(-g)) * u
    return y.to(s["x"].dtype)


_PLAIN = {"block_norm": _plain_block_norm, "block_norm_backward": _plain_block_norm_backward, "grouped_mm": _plain_grouped_mm,
          "grouped_mm_dgrad": _plain_grouped_mm_dgrad, "grouped_mm_wgrad": _plain_grouped_mm_wgrad,
          "expert_linear_w4": _plain_expert_linear_w4}


# ------------------------------------------------------------------- work ----

def work(case):
    c = case
    if c["op"].startswith("block_norm"):
        T, d = c["T"], c["d"]
        res = 4 if c["residual"] == "float32" else 2
        gate = {"none": 0, "token": T, "channel": d, "full": T * d}[c["gate"]]
        vectors = (c["post"] + c["pre"]) * d
        if c["op"] == "block_norm":
            return {"bytes": T * d * (2 + 2 * res + 2 * c["pre"]) + 2 * gate + 2 * vectors, "flops": 12.0 * T * d}
        grads = 4 * vectors + (2 if c["gate"] == "full" else 4) * gate
        # reads: y, the residual's gradient, and for the norm before the next block its gradient and the residual
        return {"bytes": T * d * (2 + 2 + 2 * res + c["pre"] * (2 + res)) + 2 * gate + 2 * vectors + grads, "flops": 30.0 * T * d}
    K, E, d, N = c["K"], c["E"], c["d"], c["N"]
    rows = c["T"] * K
    p = 1.0 / torch.arange(1, E + 1, dtype=torch.float64) ** (1.2 if c["dist"] == "zipf" else 0.0)
    p /= p.sum()
    used = min(float(E), float(rows), float((1 - (1 - p).clamp_min(0) ** rows).sum()))  # experts that some slot takes, about
    used = max(used, min(E, K))
    if c["op"].startswith("grouped_mm"):
        weights = E if c["op"] == "grouped_mm_wgrad" else used
        return {"bytes": 2.0 * (rows * (d + N) + weights * d * N), "flops": 2.0 * rows * d * N}
    out = N // 2 if c["act"] == "swiglu" else N
    per_group = 2 + (1 if c["zeros"] else 0)
    return {"bytes": used * N * (d / 2 + d // c["group"] * per_group) + 2.0 * (c["T"] * d * (K if c["per_slot"] else 1) + rows * out) + 4 * rows,
            "flops": 2.0 * rows * d * N}


# ------------------------------------------------------------------ exact ----

def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    f = lambda t: None if t is None else t.double()  # noqa: E731
    if op.startswith("block_norm"):
        y, w_post, w_pre, gate = (f(s[k]) for k in ("y", "w_post", "w_pre", "gate"))

        def norm(v, w):
            return v / (v.pow(2).sum(1, keepdim=True) / v.shape[1] + EPS).sqrt() * w

        def branch(y, w_post, gate):
            z = norm(y, w_post) if w_post is not None else y
            return case["scale"] * z * (gate if gate is not None else 1.0)

        if op == "block_norm":
            r = f(s["residual"]) + branch(y, w_post, gate)
            return {"residual_out": r, "normed": norm(r, w_pre) if w_pre is not None else None}
        # by differentiation of the definition
        leaf = lambda t: None if t is None else t.detach().requires_grad_(True)  # noqa: E731
        r, y, w_post, w_pre, gate = (leaf(t) for t in (f(s["residual_out"]), y, w_post, w_pre, gate))
        ds, d_w_pre = f(s["d_residual_out"]), None
        if w_pre is not None:
            by_r, d_w_pre = torch.autograd.grad(norm(r, w_pre), [r, w_pre], f(s["d_normed"]))
            ds = ds + by_r
        wanted = [("d_y", y), ("d_w_post", w_post), ("d_gate", gate)]
        got = torch.autograd.grad(branch(y, w_post, gate), [t for _, t in wanted if t is not None], ds)
        names = [n for n, t in wanted if t is not None]
        return {"d_residual": ds, "d_w_pre": d_w_pre, "d_w_post": None, "d_gate": None, **dict(zip(names, got))}
    if op.startswith("grouped_mm"):
        if op == "grouped_mm_wgrad":
            out = torch.zeros((case["E"], case["N"], case["d"]), dtype=torch.float64, device="cuda")
        else:
            rows = s["x" if op == "grouped_mm" else "dy"]
            out = torch.zeros((rows.shape[0], case["N" if op == "grouped_mm" else "d"]), dtype=torch.float64, device="cuda")
        for e in range(case["E"]):
            lo, hi = int(s["seg_start"][e]), int(s["seg_start"][e + 1])
            if op == "grouped_mm":
                out[lo:hi] = torch.einsum("rk,nk->rn", f(s["x"][lo:hi]), f(s["w"][e]))
            elif op == "grouped_mm_dgrad":
                out[lo:hi] = torch.einsum("rn,nk->rk", f(s["dy"][lo:hi]), f(s["w"][e]))
            else:
                out[e] = torch.einsum("rn,rk->nk", f(s["dy"][lo:hi]), f(s["x"][lo:hi]))
        return out
    T, K, d, N, G = (case[k] for k in ("T", "K", "d", "N", "group"))
    out = torch.empty((T * K, N), dtype=torch.float64, device="cuda")
    x = s["x"] if case["per_slot"] else s["x"].unsqueeze(1).expand(T, K, d)
    x, e_of = f(x).reshape(T * K, d), s["asgn"].reshape(-1)
    for e in range(case["E"]):
        at = (e_of == e).nonzero().flatten()
        if at.numel() == 0:
            continue
        w = torch.empty((N, d), dtype=torch.float64, device="cuda")
        w[:, 0::2] = (s["w_q"][e] % 16).double()
        w[:, 1::2] = (s["w_q"][e] // 16).double()
        zero = f(s["w_zero"][e]) if s["w_zero"] is not None else torch.full((N, d // G), 8.0, dtype=torch.float64, device="cuda")
        w = (w - zero.repeat_interleave(G, 1)) * f(s["w_scale"][e]).repeat_interleave(G, 1)
        out[at] = torch.mm(x[at], w.t())
    if case["act"] == "swiglu":
        return torch.sigmoid(out[:, : N // 2]) * out[:, : N // 2] * out[:, N // 2 :]
    return out
