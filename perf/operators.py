"""Performance cases of the policy head's operators: what a policy does between its residual
stream and the token logprobs.

* ``norm``: the final RMS norm with the residual's addition, for training (with its backward)
  and for scoring (an output in 8 bits with one scale per row);
* ``dropout``: counter-based dropout and its backward, whose mask is never stored;
* ``adapters``: next-token logprobs from hidden states and the output weight with low-rank
  adapters of several requests beside it (id -1: the base model), with gradients or without;
* ``scoring8``: next-token logprobs from 8-bit hidden states and an 8-bit output weight.

A case is a dict of plain values; ``prepare`` makes its inputs on the GPU, ``run`` is one pass.
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
E4M3_MAX = 448.0
M32 = 0xFFFFFFFF


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------
def listed() -> list[dict]:
    return [
        # the scoring pass of a GRPO step (8 samples of 2048 tokens): norm into the 8-bit head
        {"name": "norm_8bit_prompts", "op": "norm", "form": "8bit", "S": 2048, "B": 8, "H": 4096, "dtype": "bf16", "wdtype": "bf16"},
        # the training pass of that step
        {"name": "norm_train", "op": "norm", "form": "train", "S": 2048, "B": 8, "H": 4096, "dtype": "bf16", "wdtype": "bf16"},
        # a small fp32 model of an odd hidden size, ragged batch
        {"name": "norm_train_odd", "op": "norm", "form": "train", "S": 257, "B": 3, "H": 1021, "dtype": "f32", "wdtype": "f32"},
        # one token of each of seven requests: latency
        {"name": "norm_8bit_tokens", "op": "norm", "form": "8bit", "S": 1, "B": 7, "H": 4096, "dtype": "f16", "wdtype": "f16"},
        # dropout on the hidden states of that training step
        {"name": "dropout_train", "op": "dropout", "S": 2048, "B": 8, "H": 4096, "dtype": "bf16", "p": 0.1},
        # a small batch of odd rows: latency
        {"name": "dropout_small", "op": "dropout", "S": 37, "B": 3, "H": 1021, "dtype": "f32", "p": 0.05},
        # GRPO training step of four adapters and the base model on one frozen output weight, about 44% response rows
        {"name": "adapters_train", "op": "adapters", "train": True, "S": 2048, "B": 8, "H": 4096, "V": 151936, "N": 4, "r": 16, "p": 0.05, "dtype": "bf16", "chunk": 1024},
        # a small fp16 model with odd sizes, every row active
        {"name": "adapters_train_odd", "op": "adapters", "train": True, "S": 130, "B": 6, "H": 1000, "V": 32003, "N": 3, "r": 12, "p": 0.0, "dtype": "f16", "chunk": 0},
        # the logprob of one new token of each of 64 requests over 16 adapters
        {"name": "adapters_tokens", "op": "adapters", "train": False, "S": 2, "B": 64, "H": 4096, "V": 151936, "N": 16, "r": 16, "p": 0.0, "dtype": "bf16", "chunk": 0},
        # the scoring pass (previous or reference policy) of a GRPO step with the 8-bit head
        {"name": "scoring8_prompts", "op": "scoring8", "S": 2048, "B": 8, "H": 4096, "V": 151936},
        # a small model with odd sizes
        {"name": "scoring8_odd", "op": "scoring8", "S": 130, "B": 3, "H": 1000, "V": 32003},
        # the logprob of one new token of each of 64 requests
        {"name": "scoring8_tokens", "op": "scoring8", "S": 2, "B": 64, "H": 4096, "V": 151936},
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    """A whole number in [lo, hi], spread over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def _shape(rng, rows_max: int, s_min: int) -> tuple[int, int]:
    B = _log_int(rng, 1, 64)
    return max(s_min, _log_int(rng, s_min, max(s_min, rows_max // B))), B


def _hidden(rng, lo: int = 64, hi: int = 4096) -> int:
    H = _log_int(rng, lo, hi)
    # real hidden sizes are multiples of 64 or 128 as often as not
    return H if rng.random() < 0.5 else max(64, H // 64 * 64)


def draw(rng) -> dict:
    op = rng.choice(["norm", "norm", "dropout", "adapters", "adapters", "scoring8"])
    if op == "norm":
        S, B = _shape(rng, 16384, 1)
        dtype = rng.choice(["bf16", "f16", "f32"])
        return {"op": op, "form": rng.choice(["train", "8bit"]), "S": S, "B": B, "H": _hidden(rng, 17, 4096), "dtype": dtype,
                "wdtype": rng.choice([dtype, "f32"])}
    if op == "dropout":
        S, B = _shape(rng, 16384, 1)
        return {"op": op, "S": S, "B": B, "H": _hidden(rng, 17, 4096), "dtype": rng.choice(["bf16", "f16", "f32"]),
                "p": round(rng.uniform(0.01, 0.6), 3)}
    S, B = _shape(rng, 8192, 2)
    H, V = _hidden(rng), _log_int(rng, 1000, 151936)
    if op == "scoring8":
        return {"op": op, "S": S, "B": B, "H": H, "V": V}
    return {"op": op, "train": rng.random() < 0.6, "S": S, "B": B, "H": H, "V": V, "N": _log_int(rng, 1, 12), "r": rng.choice([4, 8, 12, 16, 24, 32, 64]),
            "p": rng.choice([0.0, 0.05, 0.1]), "dtype": rng.choice(["bf16", "bf16", "f16"]), "chunk": rng.choice([0, 512, 1024])}


# ---------------------------------------------------------------------------
# the inputs
# ---------------------------------------------------------------------------
def _gen(seed: int) -> torch.Generator:
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g: torch.Generator, *shape: int) -> torch.Tensor:
    return torch.randn(*shape, generator=g, device="cuda")


def _rows8(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Rows in e4m3 with one fp32 scale each: amax / 448 (1 for a row of zeros)."""
    x = x.float()
    amax = x.abs().amax(-1)
    scale = torch.where(amax > 0, amax / E4M3_MAX, torch.ones_like(amax))
    return (x / scale[..., None]).to(torch.float8_e4m3fn), scale


def _head(g: torch.Generator, c: dict) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Normed hidden states [S, B, H], output weight [V, H] (fp32) and targets [B, S]: logits of a
    standard deviation of about 1.5 and next tokens that the policy finds likely, as sampled
    ones are."""
    S, B, H, V = c["S"], c["B"], c["H"], c["V"]
    target = torch.randint(0, V, (B, S), generator=g, device="cuda")
    weight = _randn(g, V, H) * (1.5 / math.sqrt(H))
    nxt = target.roll(-1, dims=1).t()  # [S, B]
    lift = 14.0 * torch.rand(S, B, 1, generator=g, device="cuda")
    hidden = _randn(g, S, B, H) + weight[nxt] * (lift / 2.25)
    return hidden, weight, target


def prepare(case: dict, seed: int) -> dict:
    c = case
    g = _gen(seed)
    if c["op"] == "norm":
        dt, wdt = DTYPES[c["dtype"]], DTYPES[c["wdtype"]]
        shape = (c["S"], c["B"], c["H"])
        st = {"case": c, "x": _randn(g, *shape).to(dt), "res": (_randn(g, *shape) * 3.0).to(dt),
              "w": (1.0 + 0.2 * _randn(g, c["H"])).to(wdt)}
        if c["form"] == "train":
            for k in ("x", "res", "w"):
                st[k].requires_grad_(True)
            st["dy"], st["dh"] = _randn(g, *shape).to(dt), _randn(g, *shape).to(dt)
        return st
    if c["op"] == "dropout":
        dt = DTYPES[c["dtype"]]
        shape = (c["S"], c["B"], c["H"])
        return {"case": c, "x": _randn(g, *shape).to(dt).requires_grad_(True), "dy": _randn(g, *shape).to(dt),
                "seed": 1_000_003 * seed + 17, "offset": seed % 97}
    hidden, weight, target = _head(g, c)
    if c["op"] == "scoring8":
        h8, hs = _rows8(hidden.to(torch.bfloat16))
        w8, ws = _rows8(weight.to(torch.bfloat16))
        return {"case": c, "h8": h8, "hs": hs, "w8": w8, "ws": ws, "target": target}
    dt = DTYPES[c["dtype"]]
    S, B, H, V, N, r = (c[k] for k in ("S", "B", "H", "V", "N", "r"))
    st = {"case": c, "hidden": hidden.to(dt), "weight": weight.to(dt), "target": target,
          "a": (_randn(g, N, r, H) / math.sqrt(H)).to(dt), "b": (_randn(g, N, V, r) * (0.5 / math.sqrt(r))).to(dt),
          # -1: the base model (the reference policy)
          "ids": torch.randint(-1, N, (B,), generator=g, device="cuda"),
          "scaling": 0.5 + torch.rand(N, generator=g, device="cuda"),
          "seed": 1_000_003 * seed + 17}
    if c["train"]:
        for k in ("hidden", "a", "b"):
            st[k].requires_grad_(True)
        # prompts of a tenth to nine tenths of the samples (none in the small case) have no gradient
        grad = _randn(g, B, S - 1)
        if c["chunk"]:
            prompt = (torch.rand(B, 1, generator=g, device="cuda") * 0.8 + 0.1) * S
            grad = torch.where(torch.arange(S - 1, device="cuda")[None] >= prompt, grad, torch.zeros_like(grad))
        st["grad"] = grad
    return st


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(state: dict):
    return (_run_own if own else _run_plain)[state["case"]["op"]](state)


def _own_norm(st):
    from rl_amd.distributed.model_utils import add_rms_norm, add_rms_norm_8bit

    if st["case"]["form"] == "8bit":
        y8, scale, h = add_rms_norm_8bit(st["x"], st["res"], st["w"], eps=1e-6)
        return {"y8": y8, "scale": scale, "h": h}
    y, h = add_rms_norm(st["x"], st["res"], st["w"], eps=1e-6)
    dx, dres, dw = torch.autograd.grad([y, h], [st["x"], st["res"], st["w"]], [st["dy"], st["dh"]])
    return {"y": y.detach(), "h": h.detach(), "dx": dx, "dres": dres, "dw": dw}


def _own_dropout(st):
    from rl_amd.distributed.model_utils import dropout

    y = dropout(st["x"], st["case"]["p"], st["seed"], offset=st["offset"])
    (dx,) = torch.autograd.grad([y], [st["x"]], [st["dy"]])
    return {"y": y.detach(), "dx": dx}


def _own_adapters(st):
    from rl_amd.distributed.model_utils import from_parallel_hidden_states_to_logprobs_with_adapters

    c = st["case"]
    lp = from_parallel_hidden_states_to_logprobs_with_adapters(
        st["hidden"], st["weight"], st["a"], st["b"], st["ids"], st["scaling"], st["target"], 0, c["V"],
        inference_only=not c["train"], chunk_size=c["chunk"] or None, dropout_p=c["p"], dropout_seed=st["seed"])
    if not c["train"]:
        return {"logprobs": lp}
    dh, da, db = torch.autograd.grad([lp], [st["hidden"], st["a"], st["b"]], [st["grad"]])
    return {"logprobs": lp.detach(), "dh": dh, "da": da, "db": db}


def _own_scoring8(st):
    from rl_amd.distributed.model_utils import from_parallel_8bit_hidden_states_to_logprobs

    return {"logprobs": from_parallel_8bit_hidden_states_to_logprobs(
        st["h8"], st["hs"], st["w8"], st["ws"], st["target"], 0, st["case"]["V"])}


_run_own = {"norm": _own_norm, "dropout": _own_dropout, "adapters": _own_adapters, "scoring8": _own_scoring8}


# ---------------------------------------------------------------------------
# the plain forms: elementary operations in 32 bits, rounded once at the end
# ---------------------------------------------------------------------------
def _plain_norm(st):
    with torch.no_grad():
        x, res, w = st["x"], st["res"], st["w"]
        h = (x.float() + res.float()).to(res.dtype)  # the residual stream, as it is stored
        h32, w32 = h.float(), w.float()
        rstd = torch.rsqrt((h32 * h32).mean(-1, keepdim=True) + 1e-6)
        n = h32 * rstd
        y = n * w32
        if st["case"]["form"] == "8bit":
            y8, scale = _rows8(y)
            return {"y8": y8, "scale": scale, "h": h}
        dy = st["dy"].float()
        wdy = w32 * dy
        dh = rstd * (wdy - n * (wdy * n).mean(-1, keepdim=True)) + st["dh"].float()
        dw = (dy * n).reshape(-1, n.shape[-1]).sum(0)
        return {"y": y.to(x.dtype), "h": h, "dx": dh.to(x.dtype), "dres": dh.to(res.dtype), "dw": dw.to(w.dtype)}


def _mulhilo(m: int, x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """High and low 32 bits of m * x (int64 tensors of 32-bit values; the product wraps modulo 2^64)."""
    p = x * m
    return (p >> 32) & M32, p & M32


def _keep(n: int, p: float, seed: int, offset: int) -> tuple[torch.Tensor, float]:
    """Which of n elements dropout keeps, and what it multiplies them by.  Elements 8 q .. 8 q + 7
    take the eight 16-bit pieces of Philox4x32-10 (Salmon et al., SC 2011) of counter (q, offset)
    and key seed, low pieces first, and are kept where the piece is at least p * 65536."""
    q = torch.arange((n + 7) // 8, device="cuda")
    seed, offset = seed & (2**64 - 1), offset & (2**64 - 1)
    c = [q & M32, q >> 32, torch.full_like(q, offset & M32), torch.full_like(q, offset >> 32)]
    k0, k1 = seed & M32, seed >> 32
    for _ in range(10):
        h0, l0 = _mulhilo(0xD2511F53, c[0])
        h1, l1 = _mulhilo(0xCD9E8D57, c[2])
        c = [h1 ^ c[1] ^ k0, l1, h0 ^ c[3] ^ k1, l0]
        k0, k1 = (k0 + 0x9E3779B9) & M32, (k1 + 0xBB67AE85) & M32
    u = torch.stack([v for w in c for v in (w & 0xFFFF, w >> 16)], -1).reshape(-1)[:n]
    T = min(65536, math.floor(p * 65536 + 0.5))
    return u >= T, (65536.0 / (65536 - T) if T < 65536 else 0.0)


def _plain_dropout(st):
    with torch.no_grad():
        x, dy = st["x"], st["dy"]
        keep, scale = _keep(x.numel(), st["case"]["p"], st["seed"], st["offset"])
        keep = keep.view(x.shape)
        zero = torch.zeros((), device="cuda")
        return {"y": torch.where(keep, x.float() * scale, zero).to(x.dtype), "dx": torch.where(keep, dy.float() * scale, zero).to(x.dtype)}


def _plain_adapters(st):
    with torch.no_grad():
        c = st["case"]
        S, B, H, V = c["S"], c["B"], c["H"], c["V"]
        hidden, w = st["hidden"].float(), st["weight"].float()
        a, b = st["a"].float(), st["b"].float()
        on = st["ids"] >= 0
        ids = st["ids"].clamp(min=0)
        s = torch.where(on, st["scaling"][ids], torch.zeros(B, device="cuda"))
        dropped, keep, scale = hidden, None, 1.0
        if c["p"] > 0:
            keep, scale = _keep(hidden.numel(), c["p"], st["seed"], 0)
            keep = keep.view(hidden.shape)
            dropped = torch.where(keep, hidden * scale, torch.zeros((), device="cuda"))
        nxt = st["target"].roll(-1, dims=1)
        lp = torch.empty(B, S - 1, device="cuda")
        if c["train"]:
            dh, da, db = torch.zeros_like(hidden), torch.zeros_like(a), torch.zeros_like(b)
        for i in range(B):
            h, d, at = hidden[:-1, i], dropped[:-1, i], ids[i : i + 1]
            ai, bi = a[at][0], b[at][0]
            u = (d @ ai.t()) * s[i]
            x = h @ w.t()
            x += u @ bi.t()
            x -= x.amax(-1, keepdim=True)
            xt = x.gather(1, nxt[i, :-1, None])
            p = x.exp_()
            z = p.sum(-1, keepdim=True)
            lp[i] = (xt - z.log())[:, 0]
            if not c["train"]:
                continue
            g = p.div_(z).neg_()
            g.scatter_add_(1, nxt[i, :-1, None], torch.ones_like(xt))
            g *= st["grad"][i][:, None]
            du = (g @ bi) * s[i]
            dd = du @ ai
            if keep is not None:
                dd = torch.where(keep[:-1, i], dd * scale, torch.zeros((), device="cuda"))
            dh[:-1, i] = g @ w + dd
            da.index_add_(0, at, (du.t() @ d)[None])
            db.index_add_(0, at, (g.t() @ u)[None])
            del g
        if not c["train"]:
            return {"logprobs": lp}
        dt = st["hidden"].dtype
        return {"logprobs": lp, "dh": dh.to(dt), "da": da.to(dt), "db": db.to(dt)}


def _plain_scoring8(st):
    with torch.no_grad():
        c = st["case"]
        w, ws = st["w8"].float(), st["ws"]
        nxt = st["target"].roll(-1, dims=1)
        lp = torch.empty(c["B"], c["S"] - 1, device="cuda")
        for i in range(c["B"]):
            x = st["h8"][:-1, i].float() @ w.t()
            x *= ws[None]
            x *= st["hs"][:-1, i, None]
            x -= x.amax(-1, keepdim=True)
            xt = x.gather(1, nxt[i, :-1, None])
            lp[i] = (xt - x.exp_().sum(-1, keepdim=True).log())[:, 0]
        return {"logprobs": lp}


_run_plain = {"norm": _plain_norm, "dropout": _plain_dropout, "adapters": _plain_adapters, "scoring8": _plain_scoring8}


# ---------------------------------------------------------------------------
# the operators' definitions in 64 bits
# ---------------------------------------------------------------------------
def _philox_u16(n: int, seed: int, offset: int) -> torch.Tensor:
    """The 16-bit pieces of the generator in n elements' order, by 16-bit limbs of the products."""
    q = torch.arange(-(-n // 8), device="cuda", dtype=torch.int64)

    def product(x, m):  # (high, low) 32 bits of x * m without a 64-bit product
        xl, xh, ml, mh = x & 0xFFFF, x >> 16, m & 0xFFFF, m >> 16
        low = xl * ml
        mid = xh * ml + (low >> 16)
        mid2 = xl * mh + (mid & 0xFFFF)
        return xh * mh + (mid >> 16) + (mid2 >> 16), ((mid2 & 0xFFFF) << 16) | (low & 0xFFFF)

    seed, offset = seed % 2**64, offset % 2**64
    x0, x1 = q % 2**32, q // 2**32
    x2, x3 = torch.zeros_like(q) + offset % 2**32, torch.zeros_like(q) + offset // 2**32
    for i in range(10):
        ka, kb = (seed % 2**32 + i * 0x9E3779B9) % 2**32, (seed // 2**32 + i * 0xBB67AE85) % 2**32
        (ha, la), (hb, lb) = product(x0, 0xD2511F53), product(x2, 0xCD9E8D57)
        x0, x1, x2, x3 = hb ^ x1 ^ ka, lb, ha ^ x3 ^ kb, la
    pieces = torch.empty(q.numel(), 8, dtype=torch.int64, device="cuda")
    for j, x in enumerate((x0, x1, x2, x3)):
        pieces[:, 2 * j], pieces[:, 2 * j + 1] = x % 65536, x // 65536
    return pieces.flatten()[:n]


def _factor(n: int, p: float, seed: int, offset: int) -> torch.Tensor:
    """Dropout's factor of each element, 64 bits."""
    T = min(65536, math.floor(p * 65536 + 0.5))
    return (_philox_u16(n, seed, offset) >= T).double() * (65536.0 / max(1, 65536 - T))


def exact(case: dict, seed: int):
    c, st = case, prepare(case, seed)
    if c["op"] == "norm":
        x, res, w = (st[k].detach().double() for k in ("x", "res", "w"))
        h = (x + res).to(st["res"].dtype).double().requires_grad_(True)
        w.requires_grad_(True)
        y = h / (h.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w
        if c["form"] == "8bit":
            y = y.detach()
            scale = y.abs().amax(-1) / E4M3_MAX
            return {"y8": y / scale[..., None], "scale": scale, "h": h.detach()}
        dh, dw = torch.autograd.grad([y], [h, w], [st["dy"].double()])
        dh = dh + st["dh"].double()
        return {"y": y.detach(), "h": h.detach(), "dx": dh, "dres": dh, "dw": dw}
    if c["op"] == "dropout":
        f = _factor(st["x"].numel(), c["p"], st["seed"], st["offset"]).view(st["x"].shape)
        return {"y": st["x"].detach().double() * f, "dx": st["dy"].double() * f}
    nxt = st["target"].roll(-1, dims=1)
    lp = torch.empty(c["B"], c["S"] - 1, dtype=torch.float64, device="cuda")
    if c["op"] == "scoring8":
        w = st["w8"].double() * st["ws"].double()[:, None]
        h = st["h8"].double() * st["hs"].double()[..., None]
        for i in range(c["B"]):
            x = h[:-1, i] @ w.t()
            lp[i] = x.gather(1, nxt[i, :-1, None])[:, 0] - torch.logsumexp(x, -1)
        return {"logprobs": lp}
    h = st["hidden"].detach().double()
    f = _factor(h.numel(), c["p"], st["seed"], 0).view(h.shape) if c["p"] > 0 else None
    w = st["weight"].double()
    a, b = st["a"].detach().double(), st["b"].detach().double()
    ids, scaling = st["ids"].tolist(), st["scaling"].double()
    if c["train"]:
        dh, da, db = torch.zeros_like(h), torch.zeros_like(a), torch.zeros_like(b)
    for i, at in enumerate(ids):
        hi = h[:-1, i].clone().requires_grad_(c["train"])
        x = hi @ w.t()
        leaves = [hi]
        if at >= 0:
            ai, bi = a[at].clone().requires_grad_(c["train"]), b[at].clone().requires_grad_(c["train"])
            leaves += [ai, bi]
            d = hi if f is None else hi * f[:-1, i]
            x = x + scaling[at] * (d @ ai.t()) @ bi.t()
        rows = x.gather(1, nxt[i, :-1, None])[:, 0] - torch.logsumexp(x, -1)
        lp[i] = rows.detach()
        if c["train"]:
            grads = torch.autograd.grad([rows], leaves, [st["grad"][i].double()])
            dh[:-1, i] = grads[0]
            if at >= 0:
                da[at] += grads[1]
                db[at] += grads[2]
        del x, rows
    if not c["train"]:
        return {"logprobs": lp}
    return {"logprobs": lp, "dh": dh, "da": da, "db": db}


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case: dict) -> dict:
    c = case
    size = {"bf16": 2, "f16": 2, "f32": 4}
    if c["op"] in ("norm", "dropout"):
        n, e = c["S"] * c["B"] * c["H"], size[c["dtype"]]
        if c["op"] == "dropout":  # x and dy in, y and dx out
            return {"bytes": 4 * n * e, "flops": 2 * n}
        if c["form"] == "8bit":  # x and the residual in, the stream and the 8-bit rows out
            return {"bytes": n * (3 * e + 1) + 4 * c["S"] * c["B"], "flops": 6 * n}
        # forward as above with y in the type; backward: dy, the stream and its gradient in, two gradients out
        return {"bytes": 9 * n * e, "flops": 16 * n}
    R, H, V = (c["S"] - 1) * c["B"], c["H"], c["V"]
    if c["op"] == "scoring8":
        return {"bytes": V * (H + 4) + R * (H + 4 + 8 + 4), "flops": 2 * R * V * H}
    N, r, e = c["N"], c["r"], size[c["dtype"]]
    used = min(N, c["B"])
    inputs = V * H * e + R * (H * e + 12) + used * r * (V + H) * e
    forward = 2 * R * V * (H + r) + 2 * R * H * r
    if not c["train"]:
        return {"bytes": inputs, "flops": forward}
    active = R if not c["chunk"] else R // 2
    # dH and the adapters' gradients from the logits' gradient
    return {"bytes": inputs + R * H * e + N * r * (V + H) * e, "flops": forward + 2 * active * V * (H + 2 * r) + 4 * active * H * r}
