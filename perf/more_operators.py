"""Operators of a decoder that is served in few bits: matrices in 8-bit integers around attention over a cache in 4 bits, as cases that can be timed and compared.

  i8      y = x W': int8 weights with a scale for each output, activations rounded to int8 with a scale for each token
          (pib_gemv_fused, pib_quantize_act + pib_gemv, pib_quantize_act_rows + pib_gemm on weights of type PIB_TYPE_I8)
  cache   keys and values rounded to 4 bits on their way into the cells of a cache, and the values that those cells then stand for (pib_kv4_write, pib_kv4_read)
  attn    attention of ragged sequences over such a cache, by pages (pib_kv4_attn)

`own` chooses between the library's calls and the plain form: elementary torch operations on the same inputs.
"""
import math
import random

import torch

own = False

PAGE, GROUP = 64, 32                            # cells of a page; neighbouring channels that share a step and a lowest value
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def listed():
    return [
        # query | key | value projection of the 1.1B-shaped draft, one token: the smallest call, all latency
        {"name": "i8_qkv_draft_b1", "kind": "i8", "N": 2560, "K": 2048, "b": 1},
        # gate | up of the 70B-shaped target, a verification batch of four tokens: the call that reads most weights
        {"name": "i8_gate_up_b4", "kind": "i8", "N": 57344, "K": 8192, "b": 4},
        # neither size a multiple of a tile, a short prompt
        {"name": "i8_odd_40", "kind": "i8", "N": 21999, "K": 5700, "b": 40},
        # a long prompt of ragged length through a 28672 x 8192 matrix: the most operations
        {"name": "i8_prompt_1999", "kind": "i8", "N": 28672, "K": 8192, "b": 1999},
        # one decoded token's keys and values of a 70B-shaped layer
        {"name": "cache_b1", "kind": "cache", "type": "f32", "kv_heads": 8, "dim": 128, "tokens": 1, "pages": 64},
        # a batch of decoded tokens, heads of 64
        {"name": "cache_odd_b37", "kind": "cache", "type": "f32", "kv_heads": 4, "dim": 64, "tokens": 37, "pages": 200},
        # a portion of prompts in bfloat16
        {"name": "cache_4000", "kind": "cache", "type": "bf16", "kv_heads": 8, "dim": 128, "tokens": 4000, "pages": 300},
        # one token of the 1.1B-shaped draft behind a few hundred: the smallest attention, all latency
        {"name": "attn_draft_b1", "kind": "attn", "type": "f32", "heads": 32, "kv_heads": 4, "dim": 64, "seqs": 1, "tokens": 1, "longest": 300, "window": 0},
        # one token of a 70B-shaped layer behind a very long document
        {"name": "attn_long_b1", "kind": "attn", "type": "bf16", "heads": 64, "kv_heads": 8, "dim": 128, "seqs": 1, "tokens": 1, "longest": 131071, "window": 0},
        # a decode batch of sequences of all lengths
        {"name": "attn_ragged_b32", "kind": "attn", "type": "f32", "heads": 64, "kv_heads": 8, "dim": 128, "seqs": 32, "tokens": 1, "longest": 8190, "window": 0},
        # verification of four drafted tokens for each of sixteen sequences
        {"name": "attn_verify_b64", "kind": "attn", "type": "bf16", "heads": 64, "kv_heads": 8, "dim": 128, "seqs": 16, "tokens": 4, "longest": 5000, "window": 0},
        # portions of prompts behind what the cache holds of them already
        {"name": "attn_prompt_1999", "kind": "attn", "type": "bf16", "heads": 64, "kv_heads": 8, "dim": 128, "seqs": 2, "tokens": 1999, "longest": 4100, "window": 0},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["i8", "i8", "cache", "attn", "attn", "attn"])
    if kind == "i8":
        while True:
            N, K, b = _log(rng, 64, 57344), _log(rng, 100, 28672), rng.choice([rng.randint(1, 16), _log(rng, 1, 1999)])
            if rng.random() < 0.6:
                N, K = (N + 127) // 128 * 128, (K + 127) // 128 * 128
            if N * K <= 57344 * 8192 and N * K * b <= 28672 * 8192 * 1999 and N * b <= 28672 * 1999:
                return {"kind": "i8", "N": N, "K": K, "b": b}
    kv_heads, dim, dtype = rng.choice([1, 2, 4, 5, 8, 8, 16]), rng.choice([64, 128, 128]), rng.choice(["f32", "bf16"])
    if kind == "cache":
        tokens = rng.choice([rng.randint(1, 64), _log(rng, 1, 4000)])
        return {"kind": "cache", "type": dtype, "kv_heads": kv_heads, "dim": dim, "tokens": tokens, "pages": max(1, tokens // PAGE) * rng.randint(2, 4)}
    while True:
        c = {"kind": "attn", "type": dtype, "heads": kv_heads * rng.choice([1, 2, 4, 7, 8, 8]), "kv_heads": kv_heads, "dim": dim, "seqs": _log(rng, 1, 64),
             "tokens": rng.choice([1, 1, 1, rng.randint(2, 8), _log(rng, 9, 1999)]), "longest": _log(rng, 60, 131071), "window": rng.choice([0, 0, 0, _log(rng, 30, 4000)])}
        w, most = work(c), work({"kind": "attn", "type": "bf16", "heads": 64, "kv_heads": 8, "dim": 128, "seqs": 2, "tokens": 1999, "longest": 4100, "window": 0})
        held = sum(_lengths(c)) * kv_heads * dim
        if w["flops"] <= (most["flops"] if dtype == "bf16" else most["flops"] // 3) and held <= 131071 * 8 * 128 and c["seqs"] * c["tokens"] * c["heads"] <= 1 << 18:
            return c


def _portions(c):
    """new tokens of each sequence of an attention case; ragged where there are several"""
    r = random.Random(c["seqs"] * 7919 + c["tokens"])
    return [c["tokens"]] + [c["tokens"] if c["tokens"] <= 8 else r.randint(1, c["tokens"]) for _ in range(c["seqs"] - 1)]


def _lengths(c):
    """keys of each sequence, those of its new tokens among them"""
    r = random.Random(c["seqs"] * 104729 + c["longest"])
    return [max(n, c["longest"] if i == 0 else _log(r, max(1, c["longest"] // 50), c["longest"])) for i, n in enumerate(_portions(c))]


# ---- inputs -------------------------------------------------------------------------------------------------------------------------
def _gen(seed, salt):
    g = torch.Generator(device="cuda")
    g.manual_seed((seed * 1000003 + salt) % (1 << 62))
    return g


def _weights(c, seed):
    """int8 rows with a scale each that give outputs of about 1"""
    g = _gen(seed, 1)
    q = torch.empty(c["N"], c["K"], dtype=torch.int8, device="cuda")
    for n in range(0, c["N"], 4096):
        q[n:n + 4096] = (torch.randn(min(4096, c["N"] - n), c["K"], device="cuda", generator=g) * 36).round_().clamp_(-127, 127).to(torch.int8)
    return q, (torch.rand(c["N"], device="cuda", generator=g) + 0.5) / (36 * math.sqrt(c["K"]))


def _activations(b, K, g):
    """rows with a few channels that stand out, as activations have them"""
    x = torch.randn(b, K, device="cuda", generator=g)
    x[:, torch.randint(0, K, (max(1, K // 200),), device="cuda", generator=g)] *= 12
    return x


def _keys_values(n, c, g):
    """[n, kv_heads, dim] keys, some of whose channels lie off zero, and values"""
    H, D = c["kv_heads"], c["dim"]
    offset = torch.randn(H, D, device="cuda", generator=g) * (torch.rand(H, D, device="cuda", generator=g) < 0.1) * 3
    k = torch.randn(n, H, D, device="cuda", generator=g) + offset
    return k, torch.randn(n, H, D, device="cuda", generator=g)


def _rows(c, seed):
    """a projection's output rows, queries | keys | values, and the cells that the keys and values go to"""
    n, H, D = c["tokens"], c["kv_heads"], c["dim"]
    g = _gen(seed, 11)
    k, v = _keys_values(n, c, g)
    x = torch.cat([torch.randn(n, 2 * H * D, device="cuda", generator=g), k.reshape(n, H * D), v.reshape(n, H * D)], 1).to(TYPES[c["type"]])
    cells = torch.randperm(c["pages"] * PAGE, device="cuda", generator=g)[:n].to(torch.int32)
    return x, cells


def _sequences(c, seed):
    """queries, keys and values of all sequences one behind the other, where each one's new tokens begin, its length, its pages"""
    g = _gen(seed, 21)
    portions, lengths = _portions(c), _lengths(c)
    n = [(l + PAGE - 1) // PAGE for l in lengths]
    q = (torch.randn(sum(portions), c["heads"], c["dim"], device="cuda", generator=g) * 1.5).to(TYPES[c["type"]])
    k, v = _keys_values(sum(lengths), c, g)
    starts = torch.tensor([sum(portions[:i]) for i in range(c["seqs"] + 1)], dtype=torch.int32, device="cuda")
    lens = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    order = torch.randperm(sum(n), device="cuda", generator=g).to(torch.int32)
    pages = torch.zeros(c["seqs"], max(n), dtype=torch.int32, device="cuda")
    for i in range(c["seqs"]):
        pages[i, :n[i]] = order[sum(n[:i]):sum(n[:i + 1])]
    return q, k, v, starts, lens, pages, sum(n)


def _cells(lengths, pages):
    """the cell of every key of all sequences, one sequence behind the other"""
    return torch.cat([(pages[i, :(l + PAGE - 1) // PAGE].unsqueeze(1) * PAGE + torch.arange(PAGE, dtype=torch.int32, device="cuda")).flatten()[:l] for i, l in enumerate(lengths)])


def _half(s):
    """float64 rounded to the numbers of fp16, nearest and even, once"""
    step = ((torch.frexp(s)[1].long() - 11).clamp(min=-24) + 1023 << 52).view(torch.float64)      # a power of two, by its bits
    return torch.round(s / step) * step


def _quantised(x):
    """nibbles, steps and lowest values of groups of neighbouring channels: the latter two in fp16, quotients in 32 bits"""
    v = x.float().clamp(-60000, 60000).unflatten(-1, (-1, GROUP))
    low = v.amin(-1, keepdim=True).to(torch.float16)
    step = ((v.amax(-1, keepdim=True) - low.float()).clamp(min=0) / torch.full_like(v[..., :1], 15)).to(torch.float16)
    d = step.float()
    n = torch.where(d > 0, torch.round((v - low.float()) / torch.where(d > 0, d, 1)), 0).clamp(0, 15)
    return n.to(torch.uint8), step, low


def _held(n, step, low):
    """the values that nibbles stand for: fp16 numbers, in 32 bits"""
    return _half(low.double() + step.double() * n.double()).float().flatten(-2)


def prepare(case, seed):
    c, dev = case, "cuda"
    st = {"case": c}
    if own:
        from pipeinfer_b200 import lib as pib
        lib = st["lib"] = pib.load()
        lib.init(torch.cuda.current_device())
        st["type"] = {"f32": pib.TYPE_F32, "bf16": pib.TYPE_BF16}.get(c.get("type"))
    if c["kind"] == "i8":
        q, s = _weights(c, seed)
        st["x"] = _activations(c["b"], c["K"], _gen(seed, 2))
        if not own:
            st.update(q=q, s=s)
            return st
        st["w"] = pib.I8Weight(lib, q.data_ptr(), s.data_ptr(), c["N"], c["K"])
        st["act"] = torch.empty(lib.act_bytes(pib.TYPE_I8, c["K"], c["b"]), dtype=torch.uint8, device=dev)
        st["y"] = torch.empty(c["b"], c["N"], device=dev)
        return st
    H, D = c["kv_heads"], c["dim"]
    if c["kind"] == "cache":
        st["x"], st["cells"] = _rows(c, seed)
        st["k"], st["v"] = (torch.empty(c["tokens"], H, D, dtype=TYPES[c["type"]], device=dev) for _ in range(2))
        if own:
            st["kv"] = pib.Kv4(lib, c["pages"], H, D)
        else:
            st["held"] = [(torch.zeros(c["pages"] * PAGE, H, D // GROUP, GROUP, dtype=torch.uint8, device=dev),) + tuple(
                torch.zeros(c["pages"] * PAGE, H, D // GROUP, 1, dtype=torch.float16, device=dev) for _ in range(2)) for _ in range(2)]
        return st
    st["q"], k, v, st["starts"], st["lens"], st["pages"], n_pages = _sequences(c, seed)
    cells = _cells(_lengths(c), st["pages"])
    if not own:
        st["held"] = []
        for x in (k, v):
            st["held"].append(tuple(torch.zeros((n_pages * PAGE,) + t.shape[1:], dtype=t.dtype, device=dev).index_copy_(0, cells.long(), t) for t in _quantised(x)))
        return st
    st["kv"] = pib.Kv4(lib, n_pages, H, D)
    for i in range(0, len(cells), 4096):
        m = min(4096, len(cells) - i)
        st["kv"].write(pib.TYPE_F32, k[i:].data_ptr(), H * D, v[i:].data_ptr(), H * D, cells[i:].data_ptr(), m, torch.cuda.current_stream().cuda_stream)
    st["batch"] = pib.Kv4Batch(type=st["type"], heads=c["heads"], tokens=len(st["q"]), seqs=c["seqs"], max_tokens=max(_portions(c)), max_pages=st["pages"].shape[1], window=c["window"], scale=D ** -0.5)
    st["out"] = torch.empty_like(st["q"])
    st["scratch"] = torch.empty(st["kv"].scratch_bytes(st["batch"]), dtype=torch.uint8, device=dev)
    torch.cuda.synchronize()
    return st


# ---- one pass -----------------------------------------------------------------------------------------------------------------------
def run(st):
    c = st["case"]
    return (_own if own else _plain)[c["kind"]](st, c)


def _own_i8(st, c):
    lib, w, x, y, b, K = st["lib"], st["w"], st["x"], st["y"], c["b"], c["K"]
    s = torch.cuda.current_stream().cuda_stream
    if b <= 8 and K <= 8192:
        lib.gemv_fused(w, x.data_ptr(), b, y.data_ptr(), s)
    elif b <= 16:
        lib.quantize_act_dev(lib.TYPE_I8, x.data_ptr(), b, K, st["act"].data_ptr(), s)
        lib.gemv(w, st["act"].data_ptr(), b, y.data_ptr(), s)
    else:
        lib.quantize_act_rows(lib.TYPE_I8, x.data_ptr(), b, K, st["act"].data_ptr(), s)
        lib.gemm(w, st["act"].data_ptr(), b, y.data_ptr(), None, s)
    return y


def _own_cache(st, c):
    n, x, w = c["tokens"], st["x"], c["kv_heads"] * c["dim"]
    s = torch.cuda.current_stream().cuda_stream
    st["kv"].write(st["type"], x[:, 2 * w:].data_ptr(), x.stride(0), x[:, 3 * w:].data_ptr(), x.stride(0), st["cells"].data_ptr(), n, s)
    st["kv"].read(st["type"], st["cells"].data_ptr(), n, st["k"].data_ptr(), w, st["v"].data_ptr(), w, s)
    return st["k"], st["v"]


def _own_attn(st, c):
    w = c["heads"] * c["dim"]
    st["kv"].attention(st["batch"], st["q"].data_ptr(), w, st["starts"].data_ptr(), st["lens"].data_ptr(), st["pages"].data_ptr(), st["out"].data_ptr(), w, st["scratch"].data_ptr(),
                       torch.cuda.current_stream().cuda_stream)
    return st["out"]


def _plain_i8(st, c):
    x = st["x"]
    d = x.abs().amax(1, keepdim=True).clamp(min=2.0 ** -100) * (torch.ones((), device=x.device) / 127)
    a = torch.round(x / d).clamp(-127, 127)
    return (a @ st["q"].float().T) * (d * st["s"])


def _plain_cache(st, c):
    n, x, w, cells = c["tokens"], st["x"], c["kv_heads"] * c["dim"], st["cells"].long()
    for held, at, out in zip(st["held"], (2 * w, 3 * w), ("k", "v")):
        for whole, new in zip(held, _quantised(x[:, at:at + w].unflatten(1, (c["kv_heads"], c["dim"])))):
            whole[cells] = new
        st[out] = _held(*(t[cells] for t in held)).to(x.dtype)
    return st["k"], st["v"]


def _plain_attn(st, c):
    q, rep, portions, out = st["q"], c["heads"] // c["kv_heads"], _portions(c), torch.empty_like(st["q"])
    at = 0
    for i, (n, l) in enumerate(zip(portions, _lengths(c))):
        cells = _cells([l], st["pages"][i:i + 1]).long()
        k, v = (_held(*(t[cells] for t in held)) for held in st["held"])
        pos, key = torch.arange(l - n, l, device=q.device).unsqueeze(1), torch.arange(l, device=q.device)
        seen = (key <= pos) & (key > pos - (c["window"] or l + 1))
        for h in range(c["kv_heads"]):
            s = torch.einsum("thd,kd->htk", q[at:at + n, h * rep:(h + 1) * rep].float() * c["dim"] ** -0.5, k[:, h])
            s = torch.where(seen, s, -math.inf)
            p = torch.exp(s - s.amax(-1, keepdim=True))
            out[at:at + n, h * rep:(h + 1) * rep] = (torch.einsum("htk,kd->thd", p, v[:, h]) / p.sum(-1).T.unsqueeze(-1)).to(q.dtype)
        at += n
    return out


_own = {"i8": _own_i8, "cache": _own_cache, "attn": _own_attn}
_plain = {"i8": _plain_i8, "cache": _plain_cache, "attn": _plain_attn}


# ---- what a pass cannot do without --------------------------------------------------------------------------------------------------
def _seen(n, l, window):
    """(query, key) pairs of n new tokens at the end of l keys, and the keys that any of them sees"""
    w = window or l
    full = sum(min(l - n + i + 1, w) for i in range(n))
    return full, min(l, n - 1 + w)


def work(c):
    if c["kind"] == "i8":
        N, K, b = c["N"], c["K"], c["b"]
        return {"bytes": N * K + 4 * N + 4 * b * (N + K), "flops": 2 * b * N * K}
    size = 2 if c["type"] == "bf16" else 4
    if c["kind"] == "cache":
        values = 2 * c["tokens"] * c["kv_heads"] * c["dim"]
        # values in and out, their nibbles with a step and a lowest value for each group written and read, the cells' numbers
        return {"bytes": 2 * values * size + 2 * values * 5 // 8 + 4 * c["tokens"], "flops": 8 * values}
    pairs, keys = map(sum, zip(*(_seen(n, l, c["window"]) for n, l in zip(_portions(c), _lengths(c)))))
    return {"bytes": keys * c["kv_heads"] * c["dim"] * 2 * 5 // 8 + 2 * size * sum(_portions(c)) * c["heads"] * c["dim"] + 4 * (keys // PAGE + 2 * c["seqs"]), "flops": 4 * pairs * c["heads"] * c["dim"]}


# ---- 64-bit results from the definitions --------------------------------------------------------------------------------------------
def exact(c, seed):
    return {"i8": _exact_i8, "cache": _exact_cache, "attn": _exact_attn}[c["kind"]](c, seed)


def _exact_i8(c, seed):
    q, s = _weights(c, seed)
    x = _activations(c["b"], c["K"], _gen(seed, 2))
    # scale and quotient are 32-bit numbers by definition, rounded to the nearest each
    third = torch.tensor(1.0, device="cuda") / torch.tensor(127.0, device="cuda")
    d = torch.maximum(x.abs().max(1, keepdim=True)[0], torch.tensor(2.0 ** -100, device="cuda")) * third
    a = torch.round(x / d).double()
    y = torch.empty(c["b"], c["N"], dtype=torch.float64, device="cuda")
    for n in range(0, c["N"], 8192):
        y[:, n:n + 8192] = (a @ q[n:n + 8192].double().T) * d.double() * s[n:n + 8192].double()
    return y


def _exact_values(x):
    """what a cache holds of x [n, heads, dim], in 64 bits; steps and lowest values are fp16 numbers, differences and quotients 32-bit numbers by definition"""
    out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    for a in range(0, x.shape[-1], GROUP):
        v = x[..., a:a + GROUP].float()
        low = v.min(-1)[0].half()
        step = (v.max(-1)[0] - low.float()).div(torch.tensor(15.0, device=x.device)).half()
        n = ((v - low.float().unsqueeze(-1)) / step.float().unsqueeze(-1)).round().clamp(0, 15).double()
        e = low.double().unsqueeze(-1) + n * step.double().unsqueeze(-1)
        # to the nearest of fp16's numbers, 11 bits each and none finer than 2^-24: adding and taking away a number of the right size rounds in 64 bits
        big = (e.view(torch.int64) & (0x7ff << 52)).view(torch.float64).clamp(min=2.0 ** -14) * (1.5 * 2.0 ** 42)
        out[..., a:a + GROUP] = (e + big) - big
    return out


def _exact_cache(c, seed):
    x, _ = _rows(c, seed)
    H, D = c["kv_heads"], c["dim"]
    return _exact_values(x[:, 2 * H * D:3 * H * D].reshape(-1, H, D)), _exact_values(x[:, 3 * H * D:].reshape(-1, H, D))


def _exact_attn(c, seed):
    q, k, v, starts, lens, _, _ = _sequences(c, seed)
    starts, lens, rep = starts.tolist(), lens.tolist(), c["heads"] // c["kv_heads"]
    out, first = torch.empty(q.shape, dtype=torch.float64, device="cuda"), 0
    for i, l in enumerate(lens):
        for h in range(c["kv_heads"]):
            K, V = (_exact_values(t[first:first + l, h]) for t in (k, v))
            for t0 in range(starts[i], starts[i + 1], 256):
                t1 = min(t0 + 256, starts[i + 1])
                pos = torch.arange(t0, t1, device="cuda") + (l - starts[i + 1])
                gap = pos.unsqueeze(1) - torch.arange(l, device="cuda")
                hidden = (gap < 0) | (gap >= c["window"]) if c["window"] else gap < 0
                for r in range(h * rep, (h + 1) * rep):
                    s = (q[t0:t1, r].double() @ K.T / math.sqrt(c["dim"])).masked_fill(hidden, -math.inf)
                    out[t0:t1, r] = torch.softmax(s, 1) @ V
        first += l
    return out
