"""The two ends of a LoRA training step and its regulariser.

* Cross entropy of a linear head over a large vocabulary, from the hidden states:
  with l = x.W^T (+ s (x.A^T).B^T for a LoRA head), loss = mean over the counted
  tokens of log(sum exp l) - l[label], and its gradients of x, of A and B, and of a
  trained W.  Tokens labelled -100 are not counted.
* Embedding lookup with scaling, out[t] = c E[i_t], and the gradient of the table,
  dE[v] = c * (sum of dy[t] over the tokens with i_t = v); the padding index has none.
* Dropout whose mask comes from Philox4x32-10 (Salmon, Moraes, Dror and Shaw, 2011):
  element e takes half-word e % 8 (low half first) of the four words that the key
  (seed) makes of the counter (e // 8, call); it is kept where those 16 bits are at
  least t = rint(65536 p), and then scaled by 65536 / (65536 - t).  The LoRA linear
  with it: y = x.W0^T + drop(s (x.A^T).B^T), and its gradients.

A case runs in its plain form (elementary torch operations) where ``own`` is
False and through the framework's entry points where it is True.
"""
import math

import numpy as np
import torch

own = False

_DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_IGNORE = -100


# ------------------------------------------------------------------- cases --

def _ce(m, k, v, dt, skip, head, r=0):
    """m tokens of which the first ``skip`` are a prompt that does not count;
    head: "frozen", "trained" or "lora"."""
    return {"op": "loss", "m": m, "k": k, "v": v, "dt": dt, "skip": skip, "head": head,
            "r": r}


def listed():
    """Sizes: the hidden sizes and token counts of this repository's benchmark and
    tests (4096 features, 32000 entries, 2048 and 8192 tokens), and generic ones."""
    return [
        # one short answer behind its prompt: latency, and the head is read twice
        {"name": "loss+grad 16 tok 4096-32000", **_ce(16, 4096, 32000, "bf16", 4, "frozen")},
        # a short batch behind a frozen head
        {"name": "loss+grad 512 tok 4096-32000", **_ce(512, 4096, 32000, "bf16", 100, "frozen")},
        # ragged: odd vocabulary, few features, fp16
        {"name": "loss+grad 1001 tok 1032-50257 fp16", **_ce(1001, 1032, 50257, "fp16", 37, "frozen")},
        # an adapted head
        {"name": "loss+grad 2048 tok 4096-32000 r16", **_ce(2048, 4096, 32000, "bf16", 500, "lora", r=16)},
        # a trained head: the gradient of the whole weight too
        {"name": "loss+grad 4096 tok 2048-65536 trained", **_ce(4096, 2048, 65536, "bf16", 0, "trained")},
        # the benchmark's training batch over a large vocabulary
        {"name": "loss+grad 8192 tok 4096-128000", **_ce(8192, 4096, 128000, "bf16", 0, "frozen")},
        # a small fp32 batch into a small table: latency
        {"name": "embed 64 tok 1000x512 fp32", "op": "embed", "t": 64, "v": 1000, "d": 512,
         "dt": "fp32", "pad": 0.0},
        # a padded batch, a row length that fits no vector
        {"name": "embed 3001 tok 50257x1001 fp16", "op": "embed", "t": 3001, "v": 50257, "d": 1001,
         "dt": "fp16", "pad": 0.4},
        # the benchmark's training batch
        {"name": "embed 8192 tok 32000x4096 bf16", "op": "embed", "t": 8192, "v": 32000, "d": 4096,
         "dt": "bf16", "pad": 0.0},
        # hidden states between two layers, forward and backward
        {"name": "dropout 333x1001 fp32", "op": "drop", "m": 333, "n": 1001, "dt": "fp32", "p": 0.1},
        {"name": "dropout 8192x4096 bf16", "op": "drop", "m": 8192, "n": 4096, "dt": "bf16", "p": 0.1},
        # one LoRA layer of a training step with dropout on the adapter
        {"name": "lora 4096 tok 4096-4096 p.05", "op": "lora", "m": 4096, "k": 4096, "n": 4096, "r": 16,
         "dt": "bf16", "p": 0.05},
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["loss", "loss", "loss", "embed", "drop", "lora"])
    dt = rng.choice(["bf16", "bf16", "fp16"])
    if op == "loss":
        head = rng.choice(["frozen", "frozen", "lora", "trained"])
        m = _log_uniform(rng, 1, 8192)
        k, v = 8 * _log_uniform(rng, 16, 512), _log_uniform(rng, 1000, 128000)
        if head == "lora":
            v = (v + 7) // 8 * 8
        return _ce(m, k, v, dt, rng.randrange(m) // 2, head,
                   rng.choice([8, 16, 64]) if head == "lora" else 0)
    if op == "embed":
        return {"op": op, "t": _log_uniform(rng, 1, 16384), "v": _log_uniform(rng, 100, 65536),
                "d": _log_uniform(rng, 64, 4096), "dt": rng.choice([dt, "fp32"]),
                "pad": rng.choice([0.0, 0.0, 0.5])}
    if op == "drop":
        return {"op": op, "m": _log_uniform(rng, 1, 8192), "n": _log_uniform(rng, 64, 4096),
                "dt": rng.choice([dt, "fp32"]), "p": round(rng.uniform(0.0, 0.6), 3)}
    return {"op": op, "m": _log_uniform(rng, 8, 4096), "k": 8 * _log_uniform(rng, 16, 512),
            "n": 8 * _log_uniform(rng, 16, 512), "r": rng.choice([8, 16, 64]), "dt": dt,
            "p": round(rng.uniform(0.01, 0.3), 3)}


# --------------------------------------------------------------------- state --

def _randn(gen, *shape, scale=1.0):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32) * scale


def _rand(gen, *shape):
    return torch.rand(shape, generator=gen, device="cuda", dtype=torch.float32)


def _randint(gen, hi, *shape):
    return torch.randint(0, hi, shape, generator=gen, device="cuda")


def _adapter(gen, r, k, n, dt):
    a = ((_rand(gen, r, k) * 2 - 1) / math.sqrt(k)).to(dt)
    return a, _randn(gen, n, r, scale=0.05).to(dt)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    op, dt = case["op"], _DT[case["dt"]]
    s = {"case": case}
    if op == "loss":
        m, k, v = case["m"], case["k"], case["v"]
        w = _randn(gen, v, k, scale=1.3 / math.sqrt(k)).to(dt)
        labels = _randint(gen, v, m)
        # normalised hidden states that lean towards their label, some tokens
        # hardly and some so much that it is nearly certain
        lean = 12 * _rand(gen, m, 1)
        x = (_randn(gen, m, k) + lean * w[labels].float()).to(dt)
        labels[: case["skip"]] = _IGNORE
        s.update(x=x, w=w, labels=labels)
        wants = ["x"]
        if case["head"] == "lora":
            s["a"], s["b"] = _adapter(gen, case["r"], k, v, dt)
            s["alpha"] = 2.0 * case["r"]
            wants += ["a", "b"]
        if case["head"] == "trained":
            wants.append("w")
        for t in wants:
            s[t].requires_grad_(True)
        s["wants"] = wants
        return s
    s["seed"], s["call"] = int(_randint(gen, 1 << 62, 1)), int(_randint(gen, 1 << 20, 1))
    if op == "embed":
        t, v, d = case["t"], case["v"], case["d"]
        # token numbers as a text has them: a few are very common
        idx = (v * _rand(gen, t).double() ** 4).long().clamp(max=v - 1)
        if case["pad"]:
            idx[_rand(gen, t) < case["pad"]] = v - 1
        s.update(idx=idx, table=_randn(gen, v, d, scale=0.02).to(dt).requires_grad_(True),
                 dy=_randn(gen, t, d, scale=0.1).to(dt), scale=math.sqrt(d),
                 pad=v - 1 if case["pad"] else None)
        return s
    if op == "drop":
        m, n = case["m"], case["n"]
        s.update(x=_randn(gen, m, n).to(dt).requires_grad_(True), dy=_randn(gen, m, n, scale=0.1).to(dt))
        return s
    m, k, n, r = case["m"], case["k"], case["n"], case["r"]
    s["a"], s["b"] = _adapter(gen, r, k, n, dt)
    s.update(x=_randn(gen, m, k).to(dt), w=_randn(gen, n, k, scale=0.02).to(dt), alpha=2.0 * r,
             dy=_randn(gen, m, n, scale=0.1).to(dt))
    for t in ("x", "a", "b"):
        s[t].requires_grad_(True)
    return s


# ---------------------------------------------------------------- plain forms --

def _mul32(a, b):
    """(high, low) words of a * b, b a tensor of 32-bit words held in 64."""
    hi, lo = a >> 16, a & 0xFFFF
    return (hi * b + ((lo * b) >> 16)) >> 16, (a * b) & 0xFFFFFFFF


def _kept(n, seed, call, t, device):
    """The truth of "kept" for n elements in a row."""
    blocks = torch.arange(-(-n // 8), device=device, dtype=torch.int64)
    c0, c1 = blocks & 0xFFFFFFFF, blocks >> 32
    c2, c3 = torch.full_like(c0, call & 0xFFFFFFFF), torch.full_like(c0, call >> 32)
    k0, k1 = seed & 0xFFFFFFFF, seed >> 32
    for _ in range(10):
        h0, l0 = _mul32(0xD2511F53, c0)
        h1, l1 = _mul32(0xCD9E8D57, c2)
        c0, c1, c2, c3 = h1 ^ c1 ^ k0, l1, h0 ^ c3 ^ k1, l0
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    words = torch.stack([c0, c1, c2, c3], -1)
    return torch.stack([words & 0xFFFF, words >> 16], -1).reshape(-1)[:n] >= t


def _mask(shape, s, device):
    """What dropout multiplies by, in 32 bits."""
    t = round(65536 * s["case"]["p"])
    n = math.prod(shape)
    kept = _kept(n, s["seed"], s["call"], t, device)
    return kept.float().reshape(shape) * (65536.0 / (65536 - t))


def _plain_loss(s):
    dt = s["x"].dtype
    x, w, labels = s["x"].detach().float(), s["w"].detach().float(), s["labels"]
    lora = s["case"]["head"] == "lora"
    logits = x @ w.t()
    if lora:
        a, b = s["a"].detach().float(), s["b"].detach().float()
        sc = s["alpha"] / s["case"]["r"]
        xa = sc * (x @ a.t())
        logits += xa @ b.t()
    counted = labels != _IGNORE
    count = counted.sum()
    at = labels.clamp_min(0)[:, None]
    top = logits.max(-1, keepdim=True).values
    target = logits.gather(1, at) - top
    p = torch.exp(logits.sub_(top))
    total = p.sum(-1, keepdim=True)
    nll = (torch.log(total) - target)[:, 0]
    loss = torch.where(counted, nll, torch.zeros_like(nll)).sum() / count
    p /= total
    p.scatter_add_(1, at, torch.full_like(target, -1.0))
    p *= counted[:, None] / count
    out = [loss]
    dx = p @ w
    if lora:
        u = sc * (p @ b)
        dx += u @ a
    out.append(dx.to(dt))
    if lora:
        out += [(u.t() @ x).to(dt), (p.t() @ xa).to(dt)]
    if s["case"]["head"] == "trained":
        out.append((p.t() @ x).to(dt))
    return tuple(out)


def _plain_embed(s):
    idx, table, dy = s["idx"], s["table"].detach(), s["dy"].float()
    out = (table[idx].float() * s["scale"]).to(table.dtype)
    if s["pad"] is not None:
        dy = dy * (idx != s["pad"])[:, None]
    grad = torch.zeros(table.shape, dtype=torch.float32, device=table.device)
    grad.index_add_(0, idx, dy)
    return out, (grad * s["scale"]).to(table.dtype)


def _plain_drop(s):
    x = s["x"].detach()
    mask = _mask(x.shape, s, x.device)
    return (x.float() * mask).to(x.dtype), (s["dy"].float() * mask).to(x.dtype)


def _plain_lora(s):
    dt, sc = s["x"].dtype, s["alpha"] / s["case"]["r"]
    x, w, a, b = (s[t].detach().float() for t in ("x", "w", "a", "b"))
    dy = s["dy"].float()
    mask = _mask(dy.shape, s, dy.device)
    xa = sc * (x @ a.t())
    y = x @ w.t() + mask * (xa @ b.t())
    dz = dy * mask
    u = sc * (dz @ b)
    return y.to(dt), (dy @ w + u @ a).to(dt), (u.t() @ x).to(dt), (dz.t() @ xa).to(dt)


# -------------------------------------------------------------- framework's --

def _run_own(s):
    from metallora_b200 import ops
    op = s["case"]["op"]
    if op == "loss":
        loss = ops.linear_cross_entropy(s["x"], s["w"], s["labels"], A=s.get("a"), B=s.get("b"),
                                        alpha=s.get("alpha", 16.0), ignore_index=_IGNORE)
        return (loss.detach(), *torch.autograd.grad(loss, [s[t] for t in s["wants"]]))
    if op == "embed":
        out = ops.embedding(s["idx"], s["table"], scale=s["scale"], padding_idx=s["pad"])
        return (out.detach(), *torch.autograd.grad(out, [s["table"]], s["dy"]))
    if op == "drop":
        out = ops.dropout(s["x"], s["case"]["p"], s["seed"], call=s["call"])
        return (out.detach(), *torch.autograd.grad(out, [s["x"]], s["dy"]))
    y = ops.lora_forward(s["x"], s["w"], s["a"], s["b"], alpha=s["alpha"], dropout=s["case"]["p"],
                         training=True, dropout_seed=s["seed"], dropout_call=s["call"])
    return (y.detach(), *torch.autograd.grad(y, [s["x"], s["a"], s["b"]], s["dy"]))


def run(state):
    if own:
        return _run_own(state)
    return {"loss": _plain_loss, "embed": _plain_embed, "drop": _plain_drop,
            "lora": _plain_lora}[state["case"]["op"]](state)


def work(case):
    op, e = case["op"], 4 if case["dt"] == "fp32" else 2
    if op == "loss":
        m, k, v, r = case["m"], case["k"], case["v"], case["r"]
        counted = m - case["skip"]
        trained = case["head"] == "trained"
        adapter = r * (k + v)
        return {"bytes": e * (counted * k + m * k + v * k * (2 if trained else 1) + 2 * adapter) + 8 * m + 4,
                "flops": 2 * counted * k * v * (3 if trained else 2) + 6 * counted * adapter}
    if op == "embed":  # rows in, rows out; dy in, the table's gradient out
        t, v, d = case["t"], case["v"], case["d"]
        rows = min(t, v)
        return {"bytes": e * d * (rows + 2 * t + v) + 16 * t, "flops": 2 * t * d}
    if op == "drop":
        n = case["m"] * case["n"]
        return {"bytes": 4 * e * n, "flops": 2 * n}
    m, k, n, r = case["m"], case["k"], case["n"], case["r"]
    return {"bytes": e * (2 * m * (k + n) + n * k + 2 * r * (k + n)),
            "flops": 4 * m * n * k + 6 * m * r * (k + n)}


# ------------------------------------------------------- 64-bit definitions --

def _exact_factor(n, case, s):
    """Dropout's factors from the generator's definition, in numpy's unsigned 64 bits."""
    ctr = np.zeros((4, (n + 7) // 8), dtype=np.uint64)
    ctr[0] = np.arange(ctr.shape[1], dtype=np.uint64)
    ctr[2] = s["call"] % 2 ** 32
    ctr[3] = s["call"] // 2 ** 32
    key = [s["seed"] % 2 ** 32, s["seed"] // 2 ** 32]
    low = np.uint64(2 ** 32 - 1)
    for rnd in range(10):
        a = ctr[0] * np.uint64(0xD2511F53)
        b = ctr[2] * np.uint64(0xCD9E8D57)
        k = [np.uint64((key[0] + rnd * 0x9E3779B9) % 2 ** 32), np.uint64((key[1] + rnd * 0xBB67AE85) % 2 ** 32)]
        ctr = np.stack([(b >> np.uint64(32)) ^ ctr[1] ^ k[0], b & low,
                        (a >> np.uint64(32)) ^ ctr[3] ^ k[1], a & low])
    halves = ctr.T.astype("<u4").copy().view("<u2").reshape(-1)[:n]
    t = int(np.rint(65536 * case["p"]))
    factor = np.where(halves < t, 0.0, 65536.0 / (65536.0 - t))
    return torch.from_numpy(factor).cuda()


def _exact_loss(case, s):
    rows = (s["labels"] >= 0).nonzero()[:, 0]
    y = s["labels"][rows]
    w = s["w"].detach().double()
    lora = case["head"] == "lora"
    if lora:
        a, b = s["a"].detach().double(), s["b"].detach().double()
        sc = s["alpha"] / case["r"]
    x_all = s["x"].detach()
    dx = torch.zeros(x_all.shape, dtype=torch.float64, device="cuda")
    dw = torch.zeros_like(w) if case["head"] == "trained" else None
    da, db = (torch.zeros_like(a), torch.zeros_like(b)) if lora else (None, None)
    loss = 0.0
    for part in torch.arange(rows.numel(), device="cuda").split(1024):
        r, t = rows[part], y[part]
        x = x_all[r].double()
        z = torch.einsum("mk,vk->mv", x, w)
        if lora:
            z += sc * torch.einsum("mr,vr->mv", torch.einsum("mk,rk->mr", x, a), b)
        lse = torch.logsumexp(z, 1)
        loss = loss + (lse - z[torch.arange(len(t)), t]).sum()
        g = torch.softmax(z, 1)
        g[torch.arange(len(t)), t] -= 1
        g /= rows.numel()
        dx[r] = g.matmul(w)
        if lora:
            gb = g.matmul(b)
            dx[r] += sc * gb.matmul(a)
            da += sc * gb.T.matmul(x)
            db += sc * g.T.matmul(x.matmul(a.T))
        if dw is not None:
            dw += g.T.matmul(x)
    return (loss / rows.numel(), dx) + ((da, db) if lora else ()) + ((dw,) if dw is not None else ())


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "loss":
        return _exact_loss(case, s)
    if op == "embed":
        table, idx, c = s["table"].detach().double(), s["idx"], s["scale"]
        grad = torch.zeros_like(table)
        order = torch.argsort(idx, stable=True)
        tokens, counts = torch.unique_consecutive(idx[order], return_counts=True)
        ends = torch.cumsum(counts, 0)
        sums = torch.cumsum(s["dy"].double()[order], 0)[ends - 1]
        grad[tokens] = c * torch.diff(sums, dim=0, prepend=torch.zeros_like(sums[:1]))
        if s["pad"] is not None:
            grad[s["pad"]] = 0
        return c * table.index_select(0, idx), grad
    if op == "drop":
        x = s["x"].detach().double()
        f = _exact_factor(x.numel(), case, s).view_as(x)
        return f * x, f * s["dy"].double()
    x, w, a, b, dy = (s[t].detach().double() for t in ("x", "w", "a", "b", "dy"))
    sc = s["alpha"] / case["r"]
    f = _exact_factor(dy.numel(), case, s).view_as(dy)
    g = f * dy
    y = torch.einsum("mk,nk->mn", x, w) + f * sc * (x @ a.T @ b.T)
    return y, dy @ w + sc * (g @ b) @ a, sc * b.T @ (g.T @ x), sc * g.T @ (x @ a.T)
