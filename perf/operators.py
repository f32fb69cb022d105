"""Operators at the end of a decode step of a mixture model kept in 8-bit floating point, as cases that can be timed and compared.

  f8      y = x W': e4m3 weights with a scale for each block of 128 x 128, activations rounded to e4m3 with a scale for each 128 of a token
          (pib_gemv_fused, pib_quantize_act + pib_gemv, pib_quantize_act_rows + pib_gemm on weights of type PIB_TYPE_F8)
  moe     a whole mixture layer for 1..16 tokens: router, choice, gated experts, shared experts, residual (pib_moe_forward)
  sample  a token of each row of logits: top-k, top-p, min-p, temperature, drawn with given numbers (pib_sample)

`own` chooses between the library's calls and the plain form: elementary torch operations on the same inputs.
"""
import math

import torch

own = False

BLOCK = 128                                     # rows and columns of a weight block, columns of an activation block


def listed():
    return [
        # query | key | value projection of the 1.1B-shaped draft, one token: the smallest call, all latency
        {"name": "f8_qkv_draft_b1", "kind": "f8", "N": 2560, "K": 2048, "b": 1},
        # gate | up of the 70B-shaped target, a verification batch of four tokens: the call that reads most weights
        {"name": "f8_gate_up_b4", "kind": "f8", "N": 57344, "K": 8192, "b": 4},
        # neither size a multiple of a block, a wide verification batch
        {"name": "f8_odd_b13", "kind": "f8", "N": 21999, "K": 5700, "b": 13},
        # a short prompt through the 70B-shaped query | key | value projection
        {"name": "f8_prompt_40", "kind": "f8", "N": 10240, "K": 8192, "b": 40},
        # a long prompt of ragged length through a 28672 x 8192 matrix: the most operations
        {"name": "f8_prompt_1999", "kind": "f8", "N": 28672, "K": 8192, "b": 1999},
        # one token through many small experts, two of them shared: eight of the 66 experts' weights are read
        {"name": "moe_f8_b1", "kind": "moe", "type": "f8", "experts": 64, "top": 6, "shared": 2, "width": 2048, "ff": 1408, "b": 1, "score": "softmax", "renorm": False},
        # a full decode batch over 128 experts: most of them have a token or two
        {"name": "moe_f8_b16", "kind": "moe", "type": "f8", "experts": 128, "top": 8, "shared": 0, "width": 4096, "ff": 1536, "b": 16, "score": "softmax", "renorm": True},
        # bfloat16 experts as the layer-list models have them, a verification batch
        {"name": "moe_bf16_b4", "kind": "moe", "type": "bf16", "experts": 16, "top": 2, "shared": 1, "width": 2048, "ff": 1024, "b": 4, "score": "softmax", "renorm": True},
        # sizes that fill no block, sigmoid scores with a correction of the choice
        {"name": "moe_f8_odd_b5", "kind": "moe", "type": "f8", "experts": 10, "top": 3, "shared": 1, "width": 1000, "ff": 700, "b": 5, "score": "sigmoid", "renorm": True},
        # one sequence's next token, vocabulary of the GGUF models
        {"name": "sample_b1", "kind": "sample", "type": "f32", "rows": 1, "vocab": 32000},
        # a full batch over a large vocabulary, every row with its own settings
        {"name": "sample_b64", "kind": "sample", "type": "f32", "rows": 64, "vocab": 128256},
        # many rows of bfloat16 logits (ties), odd vocabulary
        {"name": "sample_bf16_b300", "kind": "sample", "type": "bf16", "rows": 300, "vocab": 50257},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["f8", "f8", "f8", "moe", "moe", "sample", "sample"])
    if kind == "f8":
        while True:
            N, K, b = _log(rng, 64, 57344), _log(rng, 100, 28672), rng.choice([rng.randint(1, 16), _log(rng, 1, 1999)])
            if rng.random() < 0.6:
                N, K = (N + 127) // 128 * 128, (K + 127) // 128 * 128
            if N * K <= 57344 * 8192 and N * K * b <= 28672 * 8192 * 1999 and N * b <= 28672 * 1999:
                return {"kind": "f8", "N": N, "K": K, "b": b}
    if kind == "moe":
        while True:
            t, E, D, F = rng.choice(["f8", "f8", "bf16"]), _log(rng, 4, 160), _log(rng, 256, 7168), _log(rng, 128, 4096)
            if rng.random() < 0.6:
                D, F = (D + 127) // 128 * 128, (F + 127) // 128 * 128
            c = {"kind": "moe", "type": t, "experts": E, "top": min(E, rng.randint(1, 8)), "shared": rng.choice([0, 0, 1, 2]), "width": D, "ff": F, "b": rng.randint(1, 16),
                 "score": rng.choice(["softmax", "softmax", "sigmoid"]), "renorm": rng.random() < 0.6}
            if (E + c["shared"]) * D * F * (2 if t == "bf16" else 1) <= 128 * 4096 * 1536 and c["b"] * (c["top"] + c["shared"]) * D * F <= 128 * 4096 * 1536:
                return c
    while True:
        R, V = _log(rng, 1, 300), _log(rng, 1000, 160000)
        if R * V <= 300 * 50257:
            return {"kind": "sample", "type": rng.choice(["f32", "f32", "bf16"]), "rows": R, "vocab": V}


# ---- inputs -------------------------------------------------------------------------------------------------------------------------
def _gen(seed, salt):
    g = torch.Generator(device="cuda")
    g.manual_seed((seed * 1000003 + salt) % (1 << 62))
    return g


def _blocks(n):
    return (n + BLOCK - 1) // BLOCK


def _e4m3(shape, g):
    return (torch.randn(shape, device="cuda", generator=g) * 96).clamp_(-448, 448).to(torch.float8_e4m3fn)


def _scales(shape, K, g):
    """block scales that give weights of about 1 / sqrt(K)"""
    return (torch.rand(shape, device="cuda", generator=g) + 0.5) / (96 * math.sqrt(K))


def _activations(b, K, g):
    """rows with a few channels that stand out, as activations have them"""
    x = torch.randn(b, K, device="cuda", generator=g)
    x[:, torch.randint(0, K, (max(1, K // 200),), device="cuda", generator=g)] *= 12
    return x


def _experts(c, seed):
    """[experts + shared] stacks of gate, up [ff, width] and down [width, ff]"""
    E, D, F, out = c["experts"] + c["shared"], c["width"], c["ff"], {}
    for i, (name, r, k) in enumerate((("gate", F, D), ("up", F, D), ("down", D, F))):
        g = _gen(seed, 10 + i)
        if c["type"] == "f8":
            w = torch.empty(E, r, k, dtype=torch.float8_e4m3fn, device="cuda")
            for e in range(E):
                w[e] = _e4m3((r, k), g)
            out[name + "_scales"] = _scales((E, _blocks(r), _blocks(k)), k, g)
        else:
            w = torch.empty(E, r, k, dtype=torch.bfloat16, device="cuda")
            for e in range(E):
                w[e] = torch.randn(r, k, device="cuda", generator=g) / math.sqrt(k)
        out[name] = w
    return out


SETTINGS = ((0.8, 40, 0.95, 0.05), (1.0, 0, 0.9, 0.0), (0.0, 0, 1.0, 0.0), (0.6, 20, 0.95, 0.0), (1.0, 0, 1.0, 0.0), (1.3, 0, 1.0, 0.1), (0.7, 1000, 0.8, 0.0), (1.0, 1, 0.5, 0.5))


def _logits(c, seed):
    """logits with a few likely tokens, some of them shut out (minus infinity)"""
    g = _gen(seed, 31)
    R, V = c["rows"], c["vocab"]
    l = torch.randn(R, V, device="cuda", generator=g) * 2
    l.scatter_add_(1, torch.randint(0, V, (R, 24), device="cuda", generator=g), torch.rand(R, 24, device="cuda", generator=g) * 10)
    l[:, torch.randint(0, V, (V // 100,), device="cuda", generator=g)] = -math.inf
    return l.to(torch.bfloat16 if c["type"] == "bf16" else torch.float32)


def _settings(c, seed):
    """temperature, top-k, top-p, min-p and the given number of every row"""
    R = c["rows"]
    rows = [SETTINGS[(seed + i) % len(SETTINGS)] for i in range(R)]
    t = [torch.tensor([r[j] for r in rows], dtype=torch.int32 if j == 1 else torch.float32, device="cuda") for j in range(4)]
    return t, torch.rand(R, device="cuda", generator=_gen(seed, 32))


def prepare(case, seed):
    c, kind, dev = case, case["kind"], "cuda"
    st = {"case": c}
    if kind == "f8":
        N, K, b = c["N"], c["K"], c["b"]
        g = _gen(seed, 1)
        q, s = _e4m3((N, K), g), _scales((_blocks(N), _blocks(K)), K, g)
        st["x"] = _activations(b, K, _gen(seed, 2))
        if not own:
            st.update(q=q, s=s)
            return st
        from pipeinfer_b200 import lib as pib
        lib = pib.load()
        lib.init(torch.cuda.current_device())
        st["lib"], st["w"] = lib, pib.F8Weight(lib, q.data_ptr(), s.data_ptr(), N, K)
        st["act"] = torch.empty(lib.act_bytes(pib.TYPE_F8, K, b), dtype=torch.uint8, device=dev)
        st["y"] = torch.empty(b, N, device=dev)
        return st
    if kind == "moe":
        D, E = c["width"], c["experts"]
        w = _experts(c, seed)
        g = _gen(seed, 20)
        w["router"] = torch.randn(E, D, device=dev, generator=g) / math.sqrt(D)
        w["correction"] = torch.randn(E, device=dev, generator=g) * 0.1 if c["score"] == "sigmoid" else None
        st["x"] = torch.randn(c["b"], D, device=dev, generator=g)
        st["residual"] = torch.randn(c["b"], D, device=dev, generator=g)
        if not own:
            st["w"] = w
            return st
        from pipeinfer_b200 import lib as pib
        lib = pib.load()
        lib.init(torch.cuda.current_device())
        p = {k: (v.data_ptr() if v is not None else None) for k, v in w.items()}
        st["lib"] = lib
        st["moe"] = pib.Moe(lib, pib.TYPE_F8 if c["type"] == "f8" else pib.TYPE_BF16, E, c["shared"], c["top"], D, c["ff"], score=c["score"], renorm=c["renorm"], scale=1.0, **p)
        st["scratch"] = torch.empty(st["moe"].scratch_bytes(c["b"]), dtype=torch.uint8, device=dev)
        st["y"] = torch.empty(c["b"], D, device=dev)
        return st
    st["logits"] = _logits(c, seed)
    st["settings"], st["u"] = _settings(c, seed)
    if own:
        from pipeinfer_b200 import lib as pib
        lib = pib.load()
        lib.init(torch.cuda.current_device())
        st["lib"] = lib
        t = st["settings"]
        # the rows' settings as the library's struct: temperature, top_k, top_p, min_p
        st["params"] = torch.stack([t[0], t[1].view(torch.float32), t[2], t[3]], 1).contiguous()
        st["ids"], st["p"], st["kept"] = (torch.empty(c["rows"], dtype=d, device=dev) for d in (torch.int32, torch.float32, torch.int32))
    return st


# ---- one pass -----------------------------------------------------------------------------------------------------------------------
def run(st):
    c = st["case"]
    return (_own if own else _plain)[c["kind"]](st, c)


def _own_f8(st, c):
    lib, w, x, y, b, K = st["lib"], st["w"], st["x"], st["y"], c["b"], c["K"]
    s = torch.cuda.current_stream().cuda_stream
    if b <= 8 and K <= 8192:
        lib.gemv_fused(w, x.data_ptr(), b, y.data_ptr(), s)
    elif b <= 16:
        lib.quantize_act_dev(lib.TYPE_F8, x.data_ptr(), b, K, st["act"].data_ptr(), s)
        lib.gemv(w, st["act"].data_ptr(), b, y.data_ptr(), s)
    else:
        lib.quantize_act_rows(lib.TYPE_F8, x.data_ptr(), b, K, st["act"].data_ptr(), s)
        lib.gemm(w, st["act"].data_ptr(), b, y.data_ptr(), None, s)
    return y


def _own_moe(st, c):
    st["moe"].forward(st["x"].data_ptr(), c["width"], c["b"], st["residual"].data_ptr(), c["width"], st["y"].data_ptr(), c["width"], st["scratch"].data_ptr(),
                      torch.cuda.current_stream().cuda_stream)
    return st["y"]


def _own_sample(st, c):
    lib = st["lib"]
    lib.sample(lib.TYPE_BF16 if c["type"] == "bf16" else lib.TYPE_F32, st["logits"].data_ptr(), c["vocab"], c["rows"], c["vocab"], st["params"].data_ptr(), st["u"].data_ptr(),
               st["ids"].data_ptr(), st["p"].data_ptr(), st["kept"].data_ptr(), torch.cuda.current_stream().cuda_stream)
    return st["ids"], st["p"], st["kept"]


def _spread(s, rows, cols):
    """block scales [.., nb, kb] to one for every element"""
    return s.repeat_interleave(BLOCK, -2)[..., :rows, :].repeat_interleave(BLOCK, -1)[..., :cols]


def _quantised(x):
    """rows rounded to e4m3 with a scale for each 128 columns: the values they stand for"""
    b, K = x.shape
    pad = torch.zeros(b, _blocks(K) * BLOCK, device=x.device)
    pad[:, :K] = x
    v = pad.reshape(b, -1, BLOCK)
    d = v.abs().amax(-1, keepdim=True).clamp(min=2.0 ** -100) / 448
    return ((v / d).to(torch.float8_e4m3fn).float() * d).reshape(b, -1)[:, :K]


def _plain_f8(st, c):
    return _quantised(st["x"]) @ (st["q"].float() * _spread(st["s"], c["N"], c["K"])).T


def _route(x, w, c):
    """experts of every token and their weights; choices in 64 bits, lowest index first among equals"""
    z = x.double() @ w["router"].double().T
    score = torch.softmax(z, -1) if c["score"] == "softmax" else 1 / (1 + torch.exp(-z))
    choice = score if w["correction"] is None else score + w["correction"].double()
    ids = torch.sort(choice, dim=-1, descending=True, stable=True)[1][:, :c["top"]]
    wt = torch.gather(score, 1, ids)
    if c["renorm"]:
        wt = wt / (wt.sum(-1, keepdim=True) + 1e-20)
    return ids, wt


def _plain_moe(st, c):
    x, w, E, D, F = st["x"], st["w"], c["experts"], c["width"], c["ff"]
    ids, wt = _route(x, w, c)
    shared = torch.arange(E, E + c["shared"], device=x.device)
    y = []
    for t in range(c["b"]):
        e = torch.cat([ids[t], shared])
        m = {}
        for name, r, k in (("gate", F, D), ("up", F, D), ("down", D, F)):
            m[name] = w[name].view(torch.uint8 if c["type"] == "f8" else torch.int16)[e].view(w[name].dtype).float()
            if c["type"] == "f8":
                m[name] = m[name] * _spread(w[name + "_scales"][e], r, k)
        g = m["gate"] @ x[t]
        h = g / (1 + torch.exp(-g)) * (m["up"] @ x[t])
        o = (m["down"] @ h.unsqueeze(-1)).squeeze(-1)
        f = torch.cat([wt[t].float(), torch.ones(c["shared"], device=x.device)])
        y.append(st["residual"][t] + (f.unsqueeze(-1) * o).sum(0))
    return torch.stack(y)


def _plain_sample(st, c):
    l, (temp, top_k, top_p, min_p), u = st["logits"].double(), st["settings"], st["u"]
    temp, top_p, min_p, u = (t.double().unsqueeze(1) for t in (temp, top_p, min_p, u))
    V = c["vocab"]
    order = torch.sort(l, dim=1, descending=True, stable=True)[1]
    s = torch.gather(l, 1, order)
    rel = s - s[:, :1]
    k = torch.where(top_k > 0, top_k, V).unsqueeze(1)
    rank = torch.arange(V, device=l.device).unsqueeze(0)
    keep = (rank < torch.where(temp > 0, k, 1)) & (s > -math.inf)
    w = torch.exp(rel)
    m = torch.where(keep, w, 0)
    ahead = torch.cumsum(m, 1) - m
    keep &= (top_p >= 1) | (ahead < top_p * m.sum(1, keepdim=True)) | (rank == 0)
    keep &= (w >= min_p) | (rank == 0)
    m = torch.where(keep, torch.exp(rel / torch.where(temp > 0, temp, 1)), 0)
    m = torch.zeros_like(m).scatter_(1, order, m)                       # back in the order of the vocabulary
    run_sum = torch.cumsum(m, 1)
    total = run_sum[:, -1:]
    ids = (run_sum <= u * total).sum(1).clamp(max=V - 1)
    return ids.int(), (torch.gather(m, 1, ids.unsqueeze(1)) / total).squeeze(1).float(), keep.sum(1).int()


_own = {"f8": _own_f8, "moe": _own_moe, "sample": _own_sample}
_plain = {"f8": _plain_f8, "moe": _plain_moe, "sample": _plain_sample}


# ---- what a pass cannot do without --------------------------------------------------------------------------------------------------
def work(c):
    if c["kind"] == "f8":
        N, K, b = c["N"], c["K"], c["b"]
        return {"bytes": N * K + 4 * _blocks(N) * _blocks(K) + 4 * b * (N + K), "flops": 2 * b * N * K}
    if c["kind"] == "moe":
        E, D, F, b = c["experts"], c["width"], c["ff"], c["b"]
        # experts that some token chooses, in the mean over routers
        active = E * (1 - (1 - c["top"] / E) ** b) + c["shared"]
        per = 3 * D * F * (2 if c["type"] == "bf16" else 1) + (4 * 3 * _blocks(D) * _blocks(F) if c["type"] == "f8" else 0)
        return {"bytes": int(active * per) + 4 * E * D + 12 * b * D, "flops": 2 * b * E * D + 6 * b * (c["top"] + c["shared"]) * D * F}
    R, V = c["rows"], c["vocab"]
    return {"bytes": R * V * (2 if c["type"] == "bf16" else 4) + 32 * R, "flops": 8 * R * V}


# ---- 64-bit results from the definitions --------------------------------------------------------------------------------------------
def exact(c, seed):
    return {"f8": _exact_f8, "moe": _exact_moe, "sample": _exact_sample}[c["kind"]](c, seed)


def _exact_weights(q, s, rows, cols):
    W = q.double()
    for i in range(0, rows, BLOCK):
        W[i:i + BLOCK] *= s[i // BLOCK].double().repeat_interleave(BLOCK)[:cols]
    return W


def _exact_f8(c, seed):
    N, K, b = c["N"], c["K"], c["b"]
    g = _gen(seed, 1)
    q, s = _e4m3((N, K), g), _scales((_blocks(N), _blocks(K)), K, g)
    x = _activations(b, K, _gen(seed, 2))
    a = torch.empty(b, K, dtype=torch.float64, device="cuda")
    for k in range(0, K, BLOCK):
        v = x[:, k:k + BLOCK]
        # scale and quotient are 32-bit numbers by definition, rounded to the nearest each
        d = torch.maximum(v.abs().max(1, keepdim=True)[0], torch.tensor(2.0 ** -100, device="cuda")) / 448
        a[:, k:k + BLOCK] = (v / d).to(torch.float8_e4m3fn).double() * d.double()
    y = torch.empty(b, N, dtype=torch.float64, device="cuda")
    for n in range(0, N, 64 * BLOCK):
        y[:, n:n + 64 * BLOCK] = a @ _exact_weights(q[n:n + 64 * BLOCK], s[n // BLOCK:n // BLOCK + 64], min(64 * BLOCK, N - n), K).T
    return y


def _exact_moe(c, seed):
    E, D, F, b = c["experts"], c["width"], c["ff"], c["b"]
    w = _experts(c, seed)
    g = _gen(seed, 20)
    R = (torch.randn(E, D, device="cuda", generator=g) / math.sqrt(D)).double()
    corr = (torch.randn(E, device="cuda", generator=g) * 0.1).double() if c["score"] == "sigmoid" else torch.zeros(E, dtype=torch.float64, device="cuda")
    x = torch.randn(b, D, device="cuda", generator=g).double()
    y = torch.randn(b, D, device="cuda", generator=g).double()
    z = x @ R.T
    score = (torch.exp(z - z.max(1, keepdim=True)[0]) if c["score"] == "softmax" else torch.sigmoid(z))
    if c["score"] == "softmax":
        score = score / score.sum(1, keepdim=True)
    pick = (score + corr).cpu().tolist()
    factor = torch.zeros(b, E + c["shared"], dtype=torch.float64)
    for t in range(b):
        chosen = sorted(range(E), key=lambda e: (-pick[t][e], e))[:c["top"]]
        tot = sum(float(score[t, e]) for e in chosen) + 1e-20 if c["renorm"] else 1.0
        for e in chosen:
            factor[t, e] = float(score[t, e]) / tot
        factor[t, E:] = 1
    for e in range(E + c["shared"]):
        rows = torch.nonzero(factor[:, e]).flatten().tolist()
        if not rows:
            continue
        G, U, Dn = ((_exact_weights(w[n][e], w[n + "_scales"][e], r, k) if c["type"] == "f8" else w[n][e].double()) for n, r, k in (("gate", F, D), ("up", F, D), ("down", D, F)))
        h = x[rows] @ G.T
        y[rows] += factor[rows, e].to("cuda").unsqueeze(1) * ((h * torch.sigmoid(h) * (x[rows] @ U.T)) @ Dn.T)
    return y


def _exact_sample(c, seed):
    import numpy as np
    l = _logits(c, seed).double().cpu().numpy()
    (temp, top_k, top_p, min_p), u = _settings(c, seed)
    ids, ps, kept = [], [], []
    for r in range(c["rows"]):
        T, k, P, m, ur = float(temp[r]), int(top_k[r]), float(top_p[r]), float(min_p[r]), float(u[r])
        row = l[r]
        order = np.lexsort((np.arange(len(row)), -row))
        order = order[row[order] > -np.inf]
        order = order[:1] if T <= 0 else order[:k] if k > 0 else order
        e = np.exp(row[order] - row[order[0]])
        if P < 1:
            order = order[:max(1, 1 + int(np.searchsorted(np.cumsum(e), P * e.sum(), side="left")))]
        order = order[np.exp(row[order] - row[order[0]]) >= min(m, 1.0)]
        kept.append(len(order))
        order = np.sort(order)
        e = np.exp((row[order] - row[order].max()) / (T if T > 0 else 1.0))
        run_sum = np.cumsum(e)
        i = min(int(np.searchsorted(run_sum, ur * run_sum[-1], side="right")), len(order) - 1)
        ids.append(int(order[i]))
        ps.append(e[i] / run_sum[-1])
    dev = "cuda"
    return torch.tensor(ids, dtype=torch.int32, device=dev), torch.tensor(ps, dtype=torch.float64, device=dev), torch.tensor(kept, dtype=torch.int32, device=dev)
