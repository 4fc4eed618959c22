"""Cases of the mixture-of-experts operators and of the 8-bit activation checkpoints.

Five kinds of pass:

``sort``     token slots ordered by expert
``permute``  rows sent to their experts and back with the routing weights, and both gradients
``experts``  the whole expert layer at inference: order, dispatch, gate/up, down, combine
``train``    the expert layer's training step: output and the gradients of everything
``stage``    the dense gate/up stage's training step over an 8-bit checkpoint

``own = False`` computes them with elementary torch operations in 32 bits, rounded once at the
end; ``own = True`` makes the framework's calls.  ``exact`` is the definition in 64 bits.
"""
import math

import torch

own = False

DEV = "cuda"
BF16 = torch.bfloat16


def listed():
    return [
        # one decode step of a server with 96 sequences, fine-grained experts
        dict(name="sort_decode", kind="sort", T=96, k=8, E=128, pad=0.0, skew=0.5, ids="int64"),
        # the longest prefill chunk, an eighth of it padding
        dict(name="sort_prefill", kind="sort", T=32768, k=8, E=256, pad=0.125, skew=0.5, ids="int32"),
        # a short ragged batch with padding, bf16 routing weights
        dict(name="permute_ragged", kind="permute", T=333, k=3, E=10, K=1416, pad=0.1, skew=1.0,
             ids="int64", weights="bf16"),
        # a training batch at the width of the 4096 x 14336 stage, fp32 routing weights
        dict(name="permute_train", kind="permute", T=16384, k=2, E=8, K=4096, pad=0.0, skew=0.3,
             ids="int64", weights="fp32"),
        # a single token of a chat
        dict(name="experts_one_token", kind="experts", T=1, k=2, E=8, K=4096, N=14336, pad=0.0,
             skew=0.3, ids="int64", weights="fp32"),
        # a decode batch over many small experts
        dict(name="experts_decode", kind="experts", T=64, k=8, E=64, K=2048, N=1024, pad=0.0,
             skew=0.5, ids="int64", weights="fp32"),
        # odd sizes, skewed routing, experts without rows, padding tokens
        dict(name="experts_ragged", kind="experts", T=1531, k=4, E=40, K=1416, N=712, pad=0.07,
             skew=2.0, ids="int32", weights="bf16"),
        # a prefill chunk over eight wide experts
        dict(name="experts_prefill", kind="experts", T=8192, k=2, E=8, K=4096, N=14336, pad=0.0,
             skew=0.3, ids="int64", weights="fp32"),
        # a training step over many small experts, pre-activations kept in bf16
        dict(name="train_small_experts", kind="train", T=4096, k=6, E=64, K=2048, N=1024, pad=0.0,
             skew=0.5, ids="int64", weights="bf16", checkpoint="bf16"),
        # a training step over eight wide experts, pre-activations kept in 8 bits
        dict(name="train_wide_experts", kind="train", T=8192, k=2, E=8, K=4096, N=14336, pad=0.0,
             skew=0.3, ids="int64", weights="bf16", checkpoint="e4m3"),
        # the dense stage, a short sequence with a ragged token count
        dict(name="stage_short", kind="stage", T=200, K=1024, N=2048),
        # the dense stage at the width of the 4096 x 14336 stage
        dict(name="stage_long", kind="stage", T=16384, K=4096, N=14336),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _log8(rng, lo, hi):
    return max(8, _log(rng, lo, hi) // 8 * 8)


def draw(rng):
    kind = rng.choice(["sort", "permute", "experts", "experts", "train", "stage"])
    if kind == "stage":
        while True:
            c = dict(kind=kind, T=_log(rng, 1, 16384), K=_log8(rng, 256, 8192),
                     N=_log8(rng, 256, 14336))
            if c["T"] * c["K"] * c["N"] <= 16384 * 4096 * 14336:
                return c
    while True:
        E = _log(rng, 4, 256)
        c = dict(kind=kind, T=_log(rng, 1, 32768 if kind == "sort" else 16384),
                 k=rng.randint(1, min(8, E)), E=E,
                 pad=rng.choice([0.0, rng.uniform(0.0, 0.2)]), skew=rng.uniform(0.0, 2.0),
                 ids=rng.choice(["int32", "int64"]))
        if kind == "sort":
            return c
        c.update(K=_log8(rng, 256, 8192), weights=rng.choice(["fp32", "bf16"]))
        if kind == "permute":
            if c["T"] * c["k"] * c["K"] <= 32768 * 4096:
                return c
            continue
        c.update(N=_log8(rng, 128, 14336))
        # a padded batch of the plain form stays within the largest listed case's
        if c["T"] * c["E"] * (c["K"] + 2 * c["N"]) > 8192 * 8 * 32768:
            continue
        if kind == "train":
            c.update(weights="bf16", checkpoint=rng.choice(["bf16", "e4m3"]))
        if (c["T"] * c["k"] * c["K"] * c["N"] <= 16384 * 4096 * 14336
                and c["E"] * c["K"] * c["N"] <= 8 * 4096 * 14336
                and c["T"] * c["E"] * c["K"] * c["N"] <= 8192 * 8 * 4096 * 14336):
            return c


# ---------------------------------------------------------------- inputs


def _randn(gen, *shape, std=1.0, dtype=BF16):
    t = torch.empty(shape, dtype=dtype, device=DEV).normal_(generator=gen)
    return t.mul_(std) if std != 1.0 else t


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    c = case
    T = c["T"]
    s = {"case": c}
    if c["kind"] == "stage":
        s["x"] = _randn(gen, T, c["K"])
        s["w"] = _randn(gen, c["K"], 2 * c["N"], std=c["K"] ** -0.5)
        s["dy"] = _randn(gen, T, c["N"])
        s["x"].requires_grad_(True)
        s["w"].requires_grad_(True)
        return s
    # a router: token logits on top of how popular each expert is; padding tokens have no expert
    E, k = c["E"], c["k"]
    logits = _randn(gen, T, E, dtype=torch.float32)
    logits += c["skew"] * _randn(gen, E, dtype=torch.float32)
    top, ids = logits.topk(k, dim=1)
    weights = top.softmax(dim=1)
    padding = torch.rand(T, generator=gen, device=DEV) < c["pad"]
    ids = ids.masked_fill(padding[:, None], -1)
    s["ids"] = ids.to(torch.int32 if c["ids"] == "int32" else torch.int64).contiguous()
    if c["kind"] == "sort":
        return s
    s["weights"] = weights.to(torch.float32 if c["weights"] == "fp32" else BF16).contiguous()
    # how many rows the fullest expert has: the plain form lays its products out with it
    s["fullest"] = max(1, int(torch.bincount((ids + 1).reshape(-1), minlength=E + 1)[1:].max()))
    K = c["K"]
    s["x"] = _randn(gen, T, K)
    if c["kind"] == "permute":
        s["ys"] = _randn(gen, T * k, K)
        s["gxs"] = _randn(gen, T * k, K)
        # the rows behind the last expert's are not written: the buffers hold zeros there
        s["xs_out"] = torch.zeros(T * k, K, dtype=BF16, device=DEV)
        s["gys_out"] = torch.zeros(T * k, K, dtype=BF16, device=DEV)
    else:
        s["w"] = _randn(gen, E, K, 2 * c["N"], std=K ** -0.5)
        s["w_down"] = _randn(gen, E, c["N"], K, std=c["N"] ** -0.5)
    if c["kind"] != "experts":
        s["dy"] = _randn(gen, T, K)
    if c["kind"] == "train":
        for name in ("x", "weights", "w", "w_down"):
            s[name].requires_grad_(True)
    return s


# ---------------------------------------------------------------- plain forms (32 bits)


def _plain_order(ids, E):
    flat = ids.reshape(-1).long()
    key = torch.where((flat < 0) | (flat >= E), E, flat)
    key, slot = torch.sort(key, stable=True)
    offsets = torch.searchsorted(key, torch.arange(E + 1, device=key.device))
    r = torch.arange(flat.numel(), device=key.device)
    rows = torch.empty_like(flat).scatter_(0, slot, torch.where(key < E, r, -1))
    slots = torch.where(key < E, slot, -1)
    return key, offsets, slots, rows.reshape(ids.shape)


def _plain_dispatch(x, slots, k):
    xs = x[slots.clamp(min=0) // k]
    return xs.masked_fill((slots < 0)[:, None], 0)


def _plain_combine(ys, rows, weights):
    picked = ys[rows.clamp(min=0)].masked_fill((rows < 0)[..., None], 0)
    if weights is None:
        return picked.sum(1)
    return (picked * weights[..., None]).sum(1)


class _PlainGroups:
    """Rows of each expert as one padded batch, [experts, rows, columns]; with fewer rows than
    experts, each row a batch of its own beside its expert's weights."""

    def __init__(self, key, offsets, E, fullest):
        self.alone = key.numel() <= E
        self.key, self.E = key, E
        self.valid = (key < E)[:, None]
        r = torch.arange(key.numel(), device=key.device)
        e = key.clamp(max=E - 1)
        self.e = e
        self.cap = fullest
        at = e * fullest + r - offsets[e]
        self.at = torch.where(key < E, at, E * fullest)

    def pad(self, rows):
        p = torch.zeros(self.E * self.cap + 1, rows.shape[1], device=rows.device)
        p[self.at] = rows.float().masked_fill(~self.valid, 0)
        return p[:-1].view(self.E, self.cap, -1)

    def product(self, rows, w):
        """rows[r] @ w[expert of r]"""
        if self.alone:
            y = torch.bmm(rows.float()[:, None], w[self.e].float())[:, 0]
        else:
            y = torch.bmm(self.pad(rows), w.float()).flatten(0, 1)[self.at.clamp(max=self.E * self.cap - 1)]
        return y.masked_fill(~self.valid, 0)

    def outer(self, a, g):
        """a_e^T @ g_e for each expert"""
        return torch.bmm(self.pad(a).transpose(1, 2), self.pad(g))


def _keep_8bit(v):
    """The values an 8-bit checkpoint of ``v`` stands for: e4m3 times a power of two for each
    row and 32 columns, the smallest that keeps the block's largest value at or below 448."""
    n = v.shape[1]
    b = torch.nn.functional.pad(v, (0, -n % 32)).unflatten(1, (-1, 32))
    m, x = torch.frexp(b.abs().amax(-1, keepdim=True))
    e = (x - 9 + (m > 0.875).int()).clamp(min=-127)
    q = torch.ldexp(b, -e).to(torch.float8_e4m3fn).float()
    return torch.ldexp(q, e).flatten(1)[:, :n]


def _keep(v, checkpoint):
    return _keep_8bit(v) if checkpoint == "e4m3" else v.to(BF16).float()


def _swiglu(up, gate):
    return up * gate / (1 + torch.exp(-gate))


def _swiglu_grads(dh, up, gate):
    """[grad up | grad gate]"""
    sig = 1 / (1 + torch.exp(-gate))
    return torch.cat([dh * gate * sig, dh * up * (sig + gate * sig * (1 - sig))], 1)


def _plain_stage(s):
    x, w, dy, n = s["x"].float(), s["w"].float(), s["dy"].float(), s["case"]["N"]
    up, gate = (x @ w).split(n, dim=1)
    g = _swiglu_grads(dy, _keep_8bit(up), _keep_8bit(gate))
    return _swiglu(up, gate).to(BF16), (g @ w.t()).to(BF16), (x.t() @ g).to(BF16)


def _plain_sort(s):
    _, offsets, slots, rows = _plain_order(s["ids"], s["case"]["E"])
    return offsets.int(), slots.int(), rows.int()


def _plain_permute(s):
    c = s["case"]
    key, offsets, slots, rows = _plain_order(s["ids"], c["E"])
    ok, token = slots >= 0, slots.clamp(min=0) // c["k"]
    w = s["weights"].float()
    ys, dy = s["ys"].float(), s["dy"].float()
    xs = _plain_dispatch(s["x"], slots, c["k"])
    y = _plain_combine(ys, rows, w).to(BF16)
    picked = ys[rows.clamp(min=0)].masked_fill((rows < 0)[..., None], 0)
    gw = (picked * dy[:, None]).sum(-1).to(s["weights"].dtype)
    gys = (dy[token] * w.reshape(-1)[slots.clamp(min=0), None]).masked_fill(~ok[:, None], 0).to(BF16)
    gx = _plain_combine(s["gxs"].float(), rows, None).to(BF16)
    return xs, y, gys, gw, gx


def _plain_experts(s):
    c = s["case"]
    key, offsets, slots, rows = _plain_order(s["ids"], c["E"])
    groups = _PlainGroups(key, offsets, c["E"], s["fullest"])
    xs = _plain_dispatch(s["x"].float(), slots, c["k"])
    up, gate = groups.product(xs, s["w"]).split(c["N"], dim=1)
    ys = groups.product(_swiglu(up, gate), s["w_down"])
    return _plain_combine(ys, rows, s["weights"].float()).to(BF16)


def _plain_train(s):
    c = s["case"]
    key, offsets, slots, rows = _plain_order(s["ids"], c["E"])
    groups = _PlainGroups(key, offsets, c["E"], s["fullest"])
    w_rout, dy = s["weights"].float(), s["dy"].float()
    xs = _plain_dispatch(s["x"].float(), slots, c["k"])
    up, gate = groups.product(xs, s["w"]).split(c["N"], dim=1)
    ys = groups.product(_swiglu(up, gate), s["w_down"])
    y = _plain_combine(ys, rows, w_rout)
    # backward
    picked = ys[rows.clamp(min=0)].masked_fill((rows < 0)[..., None], 0)
    g_rout = (picked * dy[:, None]).sum(-1)
    gys = dy[slots.clamp(min=0) // c["k"]] * w_rout.reshape(-1)[slots.clamp(min=0), None]
    gys = gys.masked_fill(~groups.valid, 0)
    up, gate = _keep(up, c["checkpoint"]), _keep(gate, c["checkpoint"])
    g_down = groups.outer(_swiglu(up, gate), gys)
    g = _swiglu_grads(groups.product(gys, s["w_down"].transpose(1, 2)), up, gate)
    g_w = groups.outer(xs, g)
    gx = _plain_combine(groups.product(g, s["w"].transpose(1, 2)), rows, None)
    return [t.to(BF16) for t in (y, gx, g_rout, g_w, g_down)]


# ---------------------------------------------------------------- one pass


def run(state):
    s, kind = state, state["case"]["kind"]
    if own:
        return _own(s, kind)
    with torch.no_grad():
        return {"sort": _plain_sort, "permute": _plain_permute, "experts": _plain_experts,
                "train": _plain_train, "stage": _plain_stage}[kind](s)


def _own(s, kind):
    import swiglu_fused_b200 as sg

    c = s["case"]
    if kind == "sort":
        order = sg.expert_order(s["ids"], c["E"])
        return order.offsets, order.slots, order.rows
    if kind == "permute":
        order = sg.expert_order(s["ids"], c["E"])
        xs = sg.expert_dispatch(s["x"], order, out=s["xs_out"])
        y = sg.expert_combine(s["ys"], order, s["weights"])
        gys, gw = sg.expert_combine_grad(s["dy"], s["ys"], order, s["weights"], out=s["gys_out"])
        gx = sg.expert_combine(s["gxs"], order)
        return xs, y, gys, gw, gx
    if kind == "experts":
        return sg.experts_swiglu(s["x"], s["ids"], s["weights"], s["w"], s["w_down"])
    if kind == "train":
        leaves = (s["x"], s["weights"], s["w"], s["w_down"])
        y = sg.fused_swiglu_experts(s["x"], s["ids"], s["weights"], s["w"], s["w_down"],
                                    checkpoint=c["checkpoint"])
        grads = torch.autograd.grad(y, leaves, s["dy"])
        return [y.detach(), *grads]
    h = sg.fused_swiglu(s["x"], s["w"], checkpoint="e4m3")
    return (h.detach(), *torch.autograd.grad(h, (s["x"], s["w"]), s["dy"]))


# ---------------------------------------------------------------- what a pass cannot do without


def work(case):
    c = case
    T, K = c["T"], c.get("K", 0)
    if c["kind"] == "stage":
        n = c["N"]
        # x, w, dy in; h, grad_x, grad_w out
        return {"bytes": 2.0 * (T * K + 2 * K * n + T * n + T * n + T * K + 2 * K * n),
                "flops": 3 * 2.0 * T * K * 2 * n}
    k, E = c["k"], c["E"]
    R = T * k * (1 - c["pad"])
    ids = T * k * (4 if c["ids"] == "int32" else 8)
    if c["kind"] == "sort":
        return {"bytes": float(ids + 8 * T * k + 4 * (E + 1)), "flops": float(T * k)}
    wb = 4 if c["weights"] == "fp32" else 2
    if c["kind"] == "permute":
        # x in, xs out | ys in, y out | dy, ys in, gys out | gxs in, gx out
        b = 2.0 * K * ((T + R) + (R + T) + (T + R) + (R + T)) + ids + 2 * wb * T * k
        return {"bytes": b, "flops": 2.0 * K * R * 4}
    n = c["N"]
    # the weights of the experts that are likely to have rows, were all equally popular; tokens
    # in and out
    used = E * (1 - (1 - k / E) ** max(1.0, T * (1 - c["pad"])))
    weights = 2.0 * used * (K * 2 * n + n * K)
    fwd = 2.0 * R * (K * 2 * n + n * K)
    tokens = 2.0 * 2 * T * K + ids + wb * T * k
    if c["kind"] == "experts":
        return {"bytes": weights + tokens, "flops": fwd}
    return {"bytes": 2.0 * used * 3 * K * n + 2.0 * E * 3 * K * n + tokens + 2.0 * 2 * T * K,
            "flops": 3 * fwd}


# ---------------------------------------------------------------- the definition in 64 bits


def _exact_round8(v):
    out = torch.empty_like(v)
    for j in range(0, v.shape[1], 32):
        b = v[:, j:j + 32]
        top = b.abs().amax(1, keepdim=True).clamp(min=1e-300)
        e = torch.ceil(torch.log2(top / 448))
        e = torch.where(torch.exp2(e - 1) * 448 >= top, e - 1, e)
        e = torch.where(torch.exp2(e) * 448 < top, e + 1, e).clamp(min=-127)
        scale = torch.exp2(e)
        z = b / scale
        # e4m3: three mantissa bits, smallest normal 2^-6
        step = torch.exp2(torch.floor(torch.log2(z.abs().clamp(min=2.0 ** -6))) - 3)
        out[:, j:j + 32] = torch.round(z / step) * step * scale
    return out


def _exact_grads(dh, up, gate):
    sig = torch.sigmoid(gate)
    return dh * gate * sig, dh * up * sig * (1 + gate * (1 - sig))


def exact(case, seed):
    c = case
    s = prepare(case, seed)
    if c["kind"] == "sort":
        return None
    f = {name: t.detach().double() for name, t in s.items()
         if isinstance(t, torch.Tensor) and t.is_floating_point()}
    if c["kind"] == "stage":
        n = c["N"]
        x, w = f["x"], f["w"]
        up, gate = x @ w[:, :n], x @ w[:, n:]
        h = up * gate * torch.sigmoid(gate)
        g = torch.cat(_exact_grads(f["dy"], _exact_round8(up), _exact_round8(gate)), 1)
        del up, gate
        return h, g @ w.t(), x.t() @ g
    T, k, E, K = c["T"], c["k"], c["E"], c["K"]
    ids = s["ids"].reshape(-1).tolist()
    by_expert = [[] for _ in range(E)]
    for slot, e in enumerate(ids):
        if 0 <= e < E:
            by_expert[e].append(slot)
    wr = f["weights"]
    if c["kind"] == "permute":
        xs, gys = torch.zeros_like(f["gxs"]), torch.zeros_like(f["gxs"])
        y, gx = torch.zeros_like(f["x"]), torch.zeros_like(f["x"])
        gw = torch.zeros_like(wr)
        r = 0
        for slots in by_expert:
            if not slots:
                continue
            at = torch.tensor(slots, device=DEV)
            t, j = at // k, at % k
            part = slice(r, r + len(slots))
            ws = wr[t, j][:, None]
            xs[part] = f["x"][t]
            y.index_add_(0, t, ws * f["ys"][part])
            gys[part] = ws * f["dy"][t]
            gw[t, j] = (f["dy"][t] * f["ys"][part]).sum(1)
            gx.index_add_(0, t, f["gxs"][part])
            r += len(slots)
        return xs, y, gys, gw, gx
    n = c["N"]
    y = torch.zeros(T, K, dtype=torch.float64, device=DEV)
    if c["kind"] == "train":
        gx, gr = torch.zeros_like(y), torch.zeros_like(wr)
        gw, gd = torch.zeros_like(f["w"]), torch.zeros_like(f["w_down"])
    for e, slots in enumerate(by_expert):
        if not slots:
            continue
        at = torch.tensor(slots, device=DEV)
        t, j = at // k, at % k
        x, w, wd = f["x"][t], f["w"][e], f["w_down"][e]
        up, gate = x @ w[:, :n], x @ w[:, n:]
        ye = (up * gate * torch.sigmoid(gate)) @ wd
        y.index_add_(0, t, ye * wr[t, j][:, None])
        if c["kind"] == "train":
            dy = f["dy"][t]
            gr[t, j] = (dy * ye).sum(1)
            g = dy * wr[t, j][:, None]
            if c["checkpoint"] == "e4m3":
                up, gate = _exact_round8(up), _exact_round8(gate)
            else:
                up, gate = up.float().to(BF16).double(), gate.float().to(BF16).double()
            gd[e] = (up * gate * torch.sigmoid(gate)).t() @ g
            gu, gg = _exact_grads(g @ wd.t(), up, gate)
            gw[e] = torch.cat([x.t() @ gu, x.t() @ gg], 1)
            gx.index_add_(0, t, gu @ w[:, :n].t() + gg @ w[:, n:].t())
    return y if c["kind"] == "experts" else [y, gx, gr, gw, gd]
