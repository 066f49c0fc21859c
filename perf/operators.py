"""Adapters of many requests, 8-bit activation checkpoints and layer norm, as cases that can be timed and compared.

A case is a dict of plain values; its "kind" names the operator:

  bank       one frozen projection with the adapters of many requests beside it (serving, forward)
  pack       rows of activations into 8-bit codes with a scale for each block of 32 columns, and back
  lora_bwd   the backward pass of an adapted projection whose input was kept in 8 bits
  norm_fwd   layer norm, forward
  norm_bwd   layer norm, backward: rows and the gradients of gamma and beta

Shapes are those of the repository's benchmark and tests and generic ones between and around them.  Base weights are
N(0, 0.02) in the library's storage formats, activations and gradients N(0, 1), adapters as they look early in a fine-tune.
"""
import math

import torch

own = False

DTYPE = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BLOCK = 32


def listed():
    return [
        # one sequence, one small projection: the least there is
        {"name": "bank_1024_m1", "kind": "bank", "storage": "int4", "in": 1024, "out": 1024, "m": 1, "prompts": 0,
         "adapters": 4, "rank": 16, "dtype": "bf16", "compute": "bf16"},
        # sixteen decoding sequences with twelve adapters of different ranks on the wide FFN projection
        {"name": "bank_ffn_m16", "kind": "bank", "storage": "int4", "in": 4096, "out": 14336, "m": 16, "prompts": 0,
         "adapters": 12, "rank": 32, "dtype": "bf16", "compute": "bf16"},
        # four prompts and two hundred decoding sequences in one step
        {"name": "bank_mixed_m2300", "kind": "bank", "storage": "int8", "in": 4096, "out": 4096, "m": 2300, "prompts": 4,
         "adapters": 24, "rank": 16, "dtype": "bf16", "compute": "bf16"},
        # a short fp32 batch of odd width
        {"name": "pack_f32_m37", "kind": "pack", "rows": 37, "dim": 1001, "dtype": "f32"},
        # a layer's input over a training batch (4 x 2048 tokens)
        {"name": "pack_m8192", "kind": "pack", "rows": 8192, "dim": 4096, "dtype": "bf16"},
        # the fp32 layer, small
        {"name": "lora_bwd_f32_m64", "kind": "lora_bwd", "storage": "int8", "in": 1024, "out": 1024, "m": 64, "rank": 16,
         "dtype": "f32", "compute": "f32"},
        # a short ragged batch through the down projection, int4 base
        {"name": "lora_bwd_int4_m1000", "kind": "lora_bwd", "storage": "int4", "in": 14336, "out": 4096, "m": 1000,
         "rank": 16, "dtype": "bf16", "compute": "bf16"},
        # the training shape with an int8 base: batch 4 x seq 2048
        {"name": "lora_bwd_int8_m8192", "kind": "lora_bwd", "storage": "int8", "in": 4096, "out": 4096, "m": 8192,
         "rank": 16, "dtype": "bf16", "compute": "f32"},
        # four decoding sequences
        {"name": "norm_fwd_m4", "kind": "norm_fwd", "rows": 4, "dim": 4096, "dtype": "bf16"},
        # a training batch (8 x 2048 tokens)
        {"name": "norm_fwd_m16384", "kind": "norm_fwd", "rows": 16384, "dim": 4096, "dtype": "bf16"},
        # a short fp32 batch of odd width
        {"name": "norm_bwd_f32_m333", "kind": "norm_bwd", "rows": 333, "dim": 1001, "dtype": "f32"},
        # a training batch (8 x 2048 tokens)
        {"name": "norm_bwd_m16384", "kind": "norm_bwd", "rows": 16384, "dim": 4096, "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _dim(rng, lo, hi, step=128):
    return max(lo, min(hi, step * int(round(_log(rng, lo, hi) / step))))


def draw(rng):
    kind = rng.choice(["bank", "bank", "pack", "lora_bwd", "lora_bwd", "norm_fwd", "norm_bwd"])
    case = {"kind": kind}
    if kind == "bank":
        many = rng.random() < 0.4
        case.update({"storage": rng.choice(["int4", "int8"]), "in": _dim(rng, 512, 14336), "out": _dim(rng, 512, 14336),
                     "m": _log(rng, 65, 4096) if many else _log(rng, 1, 64),
                     "prompts": rng.randint(1, 8) if many else 0, "adapters": _log(rng, 1, 64),
                     "rank": rng.choice([8, 16, 16, 32, 64]), "dtype": "bf16", "compute": "bf16"})
        if rng.random() < 0.15:
            case.update({"in": _dim(rng, 512, 2048), "out": _dim(rng, 512, 2048, 8), "m": _log(rng, 1, 64), "prompts": 0,
                         "dtype": "f32", "compute": "f32"})
        case["m"] = min(case["m"], int(1.3e11) // (case["in"] * case["out"]))
    elif kind == "lora_bwd":
        storage = rng.choice(["int4", "int8"])
        case.update({"storage": storage, "in": _dim(rng, 512, 14336), "out": _dim(rng, 512, 14336),
                     "m": _log(rng, 64, 8192), "rank": rng.choice([8, 16, 16, 32, 64]), "dtype": "bf16",
                     "compute": "f32" if storage == "int8" else "bf16"})
        if rng.random() < 0.2:
            case.update({"in": _dim(rng, 512, 2048), "out": _dim(rng, 512, 2048), "m": _log(rng, 16, 512),
                         "dtype": "f32", "compute": "f32"})
        case["m"] = min(case["m"], int(1.3e11) // (case["in"] * case["out"]))
    else:
        # (widths need not be multiples of anything)
        dim = _dim(rng, 256, 16384, 8) + rng.choice([0, 0, 0, 1, 5])
        t = rng.choice(["bf16", "bf16", "f16", "f32"])
        case.update({"rows": min(_log(rng, 1, 16384), int(3e7 if t == "f32" else 6e7) // dim), "dim": dim, "dtype": t})
    return case


# ---------------------------------------------------------------- what a program has in hand

class _Source:
    def __init__(self, seed):
        self.dev = torch.device("cuda")
        self.gen = torch.Generator(device=self.dev).manual_seed(seed)

    def normal(self, *shape, dtype=torch.bfloat16, std=1.0):
        t = torch.randn(*shape, generator=self.gen, device=self.dev)
        return (t.mul_(std) if std != 1.0 else t).to(dtype)

    def whole(self, lo, hi, n):
        return torch.randint(lo, hi, (n,), generator=self.gen, device=self.dev, dtype=torch.int32)

    def weight(self, s):
        """codes and scales of a frozen [out, in] weight: int4 two a byte with an fp16 scale per 128, or int8 with one scale"""
        w = self.normal(s["out"] * s["in"], dtype=torch.float32, std=0.02)
        if s["storage"] == "int8":
            scale = w.abs().max().div(127.0).reshape(1)
            return torch.round(w / scale).clamp_(-127, 127).to(torch.int8).view(s["out"], s["in"]), scale
        g = w.view(-1, 128)
        scale = g.abs().amax(1).div(7.0).to(torch.float16)
        q = torch.round(g / scale.float()[:, None]).clamp_(-8, 7).to(torch.int32).view(-1, 2) & 15
        return (q[:, 0] | q[:, 1] << 4).to(torch.uint8), scale


def _pack(x):
    """codes and scale bytes of the blocks of x, as the library stores them"""
    rows, dim = x.shape
    blocks = (dim + BLOCK - 1) // BLOCK
    b = torch.nn.functional.pad(x.float(), (0, blocks * BLOCK - dim)).view(rows, blocks, BLOCK)
    most = b.abs().amax(2)
    part, power = torch.frexp(most)
    e = torch.where(most > 0, power - 7 + (part * 128 > 127).int(), -126).clamp(-126, 127)
    codes = torch.round(torch.ldexp(b, -e[:, :, None])).to(torch.int8).view(rows, blocks * BLOCK)[:, :dim]
    return codes.contiguous(), (e + 127).to(torch.uint8)


def _unpack(codes, scales):
    rows, dim = codes.shape
    s = torch.ldexp(torch.ones((), device=codes.device), scales.int() - 127)
    return codes.float() * s.repeat_interleave(BLOCK, 1)[:, :dim]


def _inputs(case, seed):
    kind = case["kind"]
    src = _Source(seed)
    s = dict(case)
    t = DTYPE[case["dtype"]]
    if kind == "bank":
        n, m = case["adapters"], case["m"]
        s["codes"], s["scales"] = src.weight(case)
        # ranks as a server meets them: the largest, and smaller ones
        ranks = [max(8, case["rank"] >> (i % 3)) for i in range(n)]
        s["a"] = [src.normal(r, case["in"], dtype=t, std=1.0 / math.sqrt(case["in"])) for r in ranks]
        s["b"] = [src.normal(case["out"], r, dtype=t, std=1e-2) for r in ranks]
        s["alpha"] = [2.0 * r for r in ranks]
        # whose each of the stacked adapters' columns is, and its factor
        s["owner"] = torch.tensor([i for i, r in enumerate(ranks) for _ in range(r)], device=src.dev, dtype=torch.int32)
        s["factor"] = torch.tensor([a / r for a, r in zip(s["alpha"], ranks) for _ in range(r)], device=src.dev)
        s["x"] = src.normal(m, case["in"], dtype=t)
        # a row of a decoding sequence has any adapter or none (-1), a prompt's rows have one
        rows = src.whole(-1, n, m)
        if case["prompts"]:
            tokens = m - m // 11
            length = max(1, tokens // case["prompts"])
            at = torch.arange(m, device=src.dev) // length
            rows = torch.where(torch.arange(m, device=src.dev) < length * case["prompts"],
                               src.whole(0, n, case["prompts"])[at.clamp(max=case["prompts"] - 1)], rows)
        s["rows"] = rows
    elif kind == "pack":
        # (outliers of single columns are what blocks are for)
        s["x"] = src.normal(case["rows"], case["dim"], dtype=torch.float32)
        s["x"][:, ::97] *= 20.0
        s["x"] = s["x"].to(t)
    elif kind == "lora_bwd":
        r = case["rank"]
        s["codes"], s["scales"] = src.weight(case)
        s["a"] = src.normal(r, case["in"], dtype=t, std=1.0 / math.sqrt(case["in"]))
        s["b"] = src.normal(case["out"], r, dtype=t, std=1e-2)
        s["alpha"] = 2.0 * r
        x = src.normal(case["m"], case["in"], dtype=t)
        s["x_codes"], s["x_scales"] = _pack(x)
        s["hidden"] = (x.float() @ s["a"].float().t()).to(t)
        s["dy"] = src.normal(case["m"], case["out"], dtype=t)
    else:
        s["x"] = src.normal(case["rows"], case["dim"], dtype=torch.float32, std=1.5).add_(0.25).to(t)
        s["gamma"] = 1.0 + src.normal(case["dim"], dtype=torch.float32, std=0.1)
        s["beta"] = src.normal(case["dim"], dtype=torch.float32, std=0.1)
        if kind == "norm_bwd":
            s["dy"] = src.normal(case["rows"], case["dim"], dtype=t)
            # kept by the forward pass
            x = s["x"].double()
            s["mean"] = x.mean(1).float()
            s["rstd"] = (1.0 / torch.sqrt(x.var(1, unbiased=False) + 1e-5)).float()
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:
        _handles(s)
    return s


# ---------------------------------------------------------------- the framework's calls

def _handles(s):
    """what a program keeps beside its tensors: the frozen weight, the adapters, the layer's scratch"""
    from caif_b200 import native as nv

    s["nv"] = nv
    kind = s["kind"]
    if kind in ("bank", "lora_bwd"):
        s["w"] = nv.Weight(s["codes"], nv.I4 if s["storage"] == "int4" else nv.I8, s["in"], s["out"], s["scales"])
        s["precision"] = nv.BF16 if s["compute"] == "bf16" else nv.F32
    if kind == "bank":
        s["bank"] = nv.LoraBank([nv.Lora(a, b, al) for a, b, al in zip(s["a"], s["b"], s["alpha"])])
        need = nv.lora_bank_workspace_bytes(s["w"], s["bank"], s["m"], s["precision"])
        s["ws"] = torch.empty(max(1, need), dtype=torch.uint8, device="cuda")
    elif kind == "lora_bwd":
        s["lora"] = nv.Lora(s["a"], s["b"], s["alpha"])
        s["packed"] = nv.PackedRows(s["x_codes"], s["x_scales"])
        need = nv.lora_bwd_packed_workspace_bytes(s["w"], s["lora"], s["m"], s["precision"])
        s["ws"] = torch.empty(max(1, need), dtype=torch.uint8, device="cuda")


def _run_own(s):
    nv, kind = s["nv"], s["kind"]
    if kind == "bank":
        return nv.lora_bank_linear_fwd(s["w"], s["bank"], s["rows"], s["x"], s["precision"], workspace=s["ws"])
    if kind == "pack":
        return nv.act_unpack(nv.act_pack(s["x"]), s["x"].dtype)
    if kind == "lora_bwd":
        return nv.lora_linear_bwd_packed(s["w"], s["lora"], s["dy"], s["packed"], s["hidden"], s["precision"],
                                         workspace=s["ws"])
    if kind == "norm_fwd":
        return nv.layernorm_fwd(s["x"], s["gamma"], s["beta"], 1e-5)
    return nv.layernorm_bwd(s["dy"], s["x"], s["mean"], s["rstd"], s["gamma"])


# ---------------------------------------------------------------- one pass

def _weight_values(s):
    """the frozen weight in 32 bits"""
    if s["storage"] == "int8":
        return s["codes"].float() * s["scales"]
    c = s["codes"].int()
    q = torch.stack((c & 15, c >> 4), 1)
    q = (q ^ 8) - 8
    return (q.view(-1, 128).float() * s["scales"].float()[:, None]).view(s["out"], s["in"])


def run(s):
    if own:
        return _run_own(s)
    kind = s["kind"]
    t = DTYPE[s["dtype"]]
    if kind == "bank":
        # every adapter's columns for every row, those of other adapters taken out
        x = s["x"].float()
        h = x @ torch.cat(s["a"]).float().t() * s["factor"]
        h = torch.where(s["rows"][:, None] == s["owner"][None, :], h, 0.0)
        return (x @ _weight_values(s).t() + h @ torch.cat(s["b"], 1).float().t()).to(t)
    if kind == "pack":
        return _unpack(*_pack(s["x"])).to(t)
    if kind == "lora_bwd":
        dy, x, a, b = s["dy"].float(), _unpack(s["x_codes"], s["x_scales"]), s["a"].float(), s["b"].float()
        g = dy * (s["alpha"] / s["rank"])
        dh = g @ b
        return (dy @ _weight_values(s) + dh @ a).to(t), (dh.t() @ x).to(t), (g.t() @ s["hidden"].float()).to(t)
    x = s["x"].float()
    if kind == "norm_fwd":
        mean = x.mean(1, keepdim=True)
        off = x - mean
        rstd = 1.0 / torch.sqrt(off.square().mean(1, keepdim=True) + 1e-5)
        return (off * rstd * s["gamma"] + s["beta"]).to(t), mean[:, 0], rstd[:, 0]
    dy = s["dy"].float()
    xh = (x - s["mean"][:, None]) * s["rstd"][:, None]
    g = dy * s["gamma"]
    dx = s["rstd"][:, None] * (g - g.mean(1, keepdim=True) - xh * (g * xh).mean(1, keepdim=True))
    return dx.to(t), (dy * xh).sum(0), dy.sum(0)


# ---------------------------------------------------------------- the definitions in 64 bits

def _exact_weight(s):
    if s["storage"] == "int8":
        return s["codes"].double() * s["scales"].double()
    flat = torch.empty(s["out"] * s["in"], dtype=torch.float64, device="cuda")
    flat[0::2] = (s["codes"] % 16).double()
    flat[1::2] = (s["codes"] // 16).double()
    flat[flat > 7] -= 16
    return (flat * s["scales"].double().repeat_interleave(128)).view(s["out"], s["in"])


def _exact_rows(codes, scales):
    wide = torch.exp2(scales.double() - 127).unsqueeze(2).expand(-1, -1, BLOCK).reshape(codes.shape[0], -1)
    return codes.double() * wide[:, :codes.shape[1]]


def exact(case, seed):
    s = _inputs(case, seed)
    kind = case["kind"]
    if kind == "bank":
        x = s["x"].double()
        y = x @ _exact_weight(s).t()
        for i, (a, b, alpha) in enumerate(zip(s["a"], s["b"], s["alpha"])):
            mine = torch.nonzero(s["rows"] == i)[:, 0]
            y[mine] += alpha / a.shape[0] * (x[mine] @ a.double().t()) @ b.double().t()
        return y
    if kind == "pack":
        out = torch.empty(case["rows"], case["dim"], dtype=torch.float64, device="cuda")
        for at in range(0, case["dim"], BLOCK):
            b = s["x"][:, at:at + BLOCK].double()
            most = b.abs().amax(1, keepdim=True).clamp(min=2.0 ** -119)
            step = torch.exp2(torch.floor(torch.log2(most)) - 6)
            step = torch.where(most > 127 * step, 2 * step, step)
            out[:, at:at + BLOCK] = torch.round(b / step) * step
        return out
    if kind == "lora_bwd":
        dy, a, b = s["dy"].double(), s["a"].double(), s["b"].double()
        k = case["rank"] * 2.0 / case["rank"]
        dh = k * (dy @ b)
        return (dy @ _exact_weight(s) + dh @ a, dh.t() @ _exact_rows(s["x_codes"], s["x_scales"]),
                k * (dy.t() @ s["hidden"].double()))
    x = s["x"].double()
    if kind == "norm_fwd":
        var, mean = torch.var_mean(x, dim=1, correction=0)
        rstd = torch.rsqrt(var + 1e-5)
        return torch.addcmul(s["beta"].double(), (x - mean[:, None]) * rstd[:, None], s["gamma"].double()), mean, rstd
    dy, mean, rstd = s["dy"].double(), s["mean"].double()[:, None], s["rstd"].double()[:, None]
    xh = (x - mean) * rstd
    g = dy * s["gamma"].double()
    n = case["dim"]
    dx = rstd / n * (n * g - g.sum(1, keepdim=True) - xh * (g * xh).sum(1, keepdim=True))
    return dx, torch.einsum("rd,rd->d", dy, xh), torch.einsum("rd->d", dy)


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    kind = case["kind"]
    e = 4 if case["dtype"] == "f32" else 2
    if kind in ("bank", "lora_bwd"):
        m, i, o, r = case["m"], case["in"], case["out"], case["rank"]
        wb = i * o * (0.5 + 2 / 128) if case["storage"] == "int4" else i * o
        if kind == "lora_bwd":
            return {"bytes": wb + e * m * (2 * i * (1 + 1 / 32) / (2 * e) + o + r + i) + 2 * e * r * (i + o),
                    "flops": 2 * m * i * o + 4 * m * r * (i + o)}
        n = case["adapters"]
        ranks = [max(8, r >> (k % 3)) for k in range(n)]
        mean = sum(ranks) / n
        # adapters that at least one row has
        alone = m if not case["prompts"] else m // 11 + case["prompts"]
        used = n * (1.0 - (1.0 - 1.0 / (n + 1)) ** alone)
        return {"bytes": wb + e * m * (i + o) + 4 * m + used * mean * e * (i + o),
                "flops": 2 * m * i * o + 2 * m * mean * (i + o)}
    rows, dim = case["rows"], case["dim"]
    if kind == "pack":
        return {"bytes": rows * dim * (2 * e + 2 * (1 + 1 / 32)), "flops": 4 * rows * dim}
    if kind == "norm_fwd":
        return {"bytes": 2 * e * rows * dim + 8 * rows + 8 * dim, "flops": 8 * rows * dim}
    return {"bytes": 3 * e * rows * dim + 8 * rows + 12 * dim, "flops": 16 * rows * dim}
