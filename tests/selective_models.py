"""Small models of selective state space layers and attention beside experts chosen by groups, and their statement in 64 bits, whole
sequences at a time (no step, no cache, none of the package's kernels)."""
import math

import torch

from inferflux_b200.config import ModelPlan, PartSpec, default_schedule, prenorm_layer

H, V, PAGE = 64, 210, 8
EPS = 1e-5


def plan(which):
    """`groups`: sigmoid scores, two of four groups, scaled weights; `softmax`: softmax scores over one best expert a group, with norms in
    front of the step, a state of 5 and a convolution of 3."""
    odd = which == "softmax"
    mixer = PartSpec("selective_state_space", {"hidden_size": H, "inner_size": 96 if odd else 128, "state_dim": 5 if odd else 16, "step_rank": 8,
                                               "conv_taps": 3 if odd else 4, "norms": odd, "norm_eps": EPS})
    if odd:
        routed = {"num_experts": 12, "top": 3, "routing": "softmax_normalized", "groups": {"count": 6, "kept": 3, "best": 1}, "correction": False,
                  "activation": "relu2", "weight_floor": 1e-9}
    else:
        routed = {"num_experts": 16, "top": 4, "routing": "sigmoid_normalized", "groups": {"count": 4, "kept": 2, "best": 2}, "weight_scale": 2.5,
                  "activation": "silu_glu", "weight_floor": 1e-20}
    ffn = PartSpec("moe", {"hidden_size": H, "expert_size": 48, **routed})
    attn = PartSpec("attention", {"hidden_size": H, "num_heads": 4, "num_kv_heads": 2, "head_dim": 16, "window": None, "qkv_bias": False,
                                  "scale": None, "position": PartSpec("rope", {"theta": 1e4, "rotary_dim": 16})})
    norm = PartSpec("rmsnorm", {"size": H, "eps": EPS})
    layers = [prenorm_layer(f"model.layers.{i}.", m, ffn, norm, norm) for i, m in enumerate((mixer, attn, mixer))]
    return ModelPlan("SelectiveHybrid", H, V, 512, PartSpec("embedding", {"vocab_size": V, "hidden_size": H}), layers, default_schedule(3), norm,
                     PartSpec("lm_head", {"vocab_size": V, "hidden_size": H, "tied": False}))


def weights(expected, seed=7):
    """Weights that make every part count: spread rates, steps and corrections, and taps."""
    from inferflux_b200.weights import random_tensors
    W = random_tensors(expected, seed=seed, dtype=torch.float32, std=0.12, norm_jitter=0.2)
    g = torch.Generator().manual_seed(seed)
    for name in sorted(W):
        if name.endswith("A_log"):
            W[name] = torch.rand(W[name].shape, generator=g) * 2.5
        elif name.endswith("dt.b"):
            W[name] = torch.rand(W[name].shape, generator=g) * 4 - 4
        elif name.endswith("correction") or name.endswith("conv.b"):
            W[name] = 0.2 * torch.randn(W[name].shape, generator=g)
        elif name.endswith(".conv"):
            W[name] = 0.4 * torch.randn(W[name].shape, generator=g)
        elif name.endswith("router"):
            W[name] = W[name] * 4
    W["model.embed_tokens.weight"] *= 8
    return W


def _rms(x, w):
    return x / (x.square().mean(-1, keepdim=True) + EPS).sqrt() * w


def _silu(v):
    return v / (1 + torch.exp(-v))


def _selective(h, W, p, params):
    C, N, R, taps = params["inner_size"], params["state_dim"], params["step_rank"], params["conv_taps"]
    xz = h @ W[p + "in"].t()
    x, z = xz[:, :C], xz[:, C:]
    padded = torch.cat([torch.zeros(taps - 1, C, dtype=x.dtype), x])
    x = _silu(sum(padded[j:j + len(h)] * W[p + "conv"][:, j] for j in range(taps)) + W[p + "conv.b"])
    s, B, Cm = (x @ W[p + "x"].t()).split([R, N, N], 1)
    if params["norms"]:
        s, B, Cm = _rms(s, W[p + "dt_norm"]), _rms(B, W[p + "b_norm"]), _rms(Cm, W[p + "c_norm"])
    step = torch.log1p(torch.exp(s @ W[p + "dt"].t() + W[p + "dt.b"]))
    state, ys = torch.zeros(C, N, dtype=x.dtype), []
    for t in range(len(h)):
        state = torch.exp(-step[t][:, None] * W[p + "A_log"].exp()) * state + step[t][:, None] * x[t][:, None] * B[t]
        ys.append(state @ Cm[t] + W[p + "D"] * x[t])
    return (torch.stack(ys) * _silu(z)) @ W[p + "o"].t()


def _attention(h, W, p, params):
    T, nq, nkv, d = len(h), 4, 2, 16
    q, k, v = (h @ W[p + f"{n}_proj.weight"].t() for n in "qkv")
    angle = torch.arange(T, dtype=h.dtype)[:, None] * (1e4 ** (-torch.arange(0, d, 2, dtype=h.dtype) / d))[None]

    def turn(r, n):
        a, b = r.view(T, n, d).split(d // 2, 2)
        c, s = angle.cos()[:, None], angle.sin()[:, None]
        return torch.cat([a * c - b * s, b * c + a * s], 2)
    q, k, v = turn(q, nq), turn(k, nkv).repeat_interleave(2, 1), v.view(T, nkv, d).repeat_interleave(2, 1)
    scores = torch.einsum("ihd,jhd->hij", q, k) * d ** -0.5
    scores = scores.masked_fill(torch.ones(T, T, dtype=torch.bool).triu(1), -math.inf)
    return torch.einsum("hij,jhd->ihd", torch.softmax(scores, 2), v).reshape(T, nq * d) @ W[p + "o_proj.weight"].t()


def _experts(h, W, p, params):
    z = h @ W[p + "router"].t()
    groups, n = params["groups"], params["num_experts"]
    score = torch.sigmoid(z) if params["routing"] == "sigmoid_normalized" else torch.softmax(z, 1)
    v = score + (W[p + "correction"] if params.get("correction", True) else 0.0)
    strength = v.view(len(h), groups["count"], -1).topk(groups["best"], 2).values.sum(2)
    kept = torch.zeros_like(strength).scatter(1, strength.topk(groups["kept"], 1).indices, 1.0).bool().repeat_interleave(n // groups["count"], 1)
    ids = v.masked_fill(~kept, -math.inf).topk(params["top"], 1).indices
    w = score.gather(1, ids)
    w = w / (w.sum(1, keepdim=True) + params["weight_floor"]) * params.get("weight_scale", 1.0)
    out = torch.zeros_like(h)
    for t in range(len(h)):
        for e, we in zip(ids[t].tolist(), w[t]):
            up = W[p + f"e{e}.up"] @ h[t]
            act = _silu(W[p + f"e{e}.gate"] @ h[t]) * up if params["activation"] == "silu_glu" else up.clamp(min=0).square()
            out[t] += we * (W[p + f"e{e}.down"] @ act)
    return out


def logits(which, W, tokens):
    W = {k: v.double() for k, v in W.items()}
    x = W["model.embed_tokens.weight"][torch.tensor(tokens)]
    for layer in plan(which).layers:
        p = layer.prefix
        mixer = _attention if layer.mixer.kind == "attention" else _selective
        x = x + mixer(_rms(x, W[p + "input_layernorm.weight"]), W, p + "self_attn.", layer.mixer.params)
        x = x + _experts(_rms(x, W[p + "post_attention_layernorm.weight"]), W, p + "mlp.", layer.ffn.params)
    return _rms(x, W["model.norm.weight"]) @ W["lm_head.weight"].t()


def made(which, dtype, device):
    """(model, the weights it was loaded with, rounded to the run's dtype where it rounds them)."""
    from inferflux_b200.models import Model
    model = Model(plan(which))
    W = weights(model.expected_tensors())
    model.load(W, dtype, device)
    if dtype != torch.float32:
        kept = ("A_log", "dt.b", "D", "correction", "conv", "conv.b", "norm", "norm.weight")
        W = {k: v if k.endswith(kept) else v.to(dtype).float() for k, v in W.items()}
    return model, W
