"""Measured cases of the attention operators over packed prompts and the paged 8-bit KV cache.

Three operators, as a serving loop runs them one after another in every layer:

append   wl_dev_rope_kv_append_i8: rotates queries and keys to their positions and appends keys and
         values to a paged int8 cache with one scale for each page and KV head.
decode   wl_dev_attn_decode_i8: attention of one token per sequence over that cache.
prompt   wl_dev_attn_prompt: causal attention of packed whole prompts, grouped heads.

Where ``own`` is false, ``run`` computes them in elementary torch operations in 32 bits; where it is
true, it calls the library.
"""
import random

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
GGML = {"f32": 0, "f16": 1, "bf16": 30}


# --------------------------------------------------------------------------------- the cases

def listed():
    return [
        # one decode step of 32 sequences at SmolLM-135M's shapes (9 query heads, 3 KV heads of 64),
        # f32 activations straight from the linears
        dict(name="append-step-smollm-32", op="append", type="f32", heads=9, kv=3, dim=64, rot=64,
             pairs=1, page=32, seqs=32, least=1, most=1, mix=1, out="f32", copies=False),
        # one decode step of 64 sequences at BitNet-2B's shapes (20 / 5 heads of 128)
        dict(name="append-step-bitnet-64", op="append", type="f32", heads=20, kv=5, dim=128, rot=128,
             pairs=0, page=64, seqs=64, least=1, most=1, mix=2, out="f16", copies=False),
        # one 512-token prompt (the prompt of the decode benchmark), f16 copies for the prompt attention
        dict(name="append-prompt-bitnet-512", op="append", type="f32", heads=20, kv=5, dim=128,
             rot=128, pairs=0, page=64, seqs=1, least=512, most=512, mix=3, out="f16", copies=True),
        # packed prompts of many lengths, bf16 model, half of each head rotated
        dict(name="append-prompts-32-heads", op="append", type="bf16", heads=32, kv=8, dim=128, rot=64,
             pairs=0, page=16, seqs=24, least=17, most=1500, mix=4, out="bf16", copies=True),
        # one sequence at the decode benchmark's last context (512 + 128): latency
        dict(name="decode-bitnet-1x640", op="decode", type="f32", heads=20, kv=5, dim=128, page=64,
             seqs=1, least=640, most=640, mix=5, out="f32"),
        # the batched decode benchmark: 32 sequences with contexts in [64, 1024]
        dict(name="decode-smollm-32x1024", op="decode", type="f32", heads=9, kv=3, dim=64, page=32,
             seqs=32, least=64, most=1024, mix=6, out="f32"),
        # a full serving batch at BitNet-2B's shapes, contexts to 8k
        dict(name="decode-bitnet-64x8k", op="decode", type="f16", heads=20, kv=5, dim=128, page=64,
             seqs=64, least=100, most=8192, mix=7, out="f16"),
        # few long contexts, 8 query heads a KV head
        dict(name="decode-long-4x100k", op="decode", type="bf16", heads=32, kv=4, dim=128, page=128,
             seqs=4, least=70001, most=100000, mix=8, out="bf16"),
        # one short chat turn
        dict(name="prompt-smollm-1x77", op="prompt", type="f16", heads=9, kv=3, dim=64, seqs=1,
             least=77, most=77, mix=9),
        # 32 packed prompts of the batched benchmark's lengths
        dict(name="prompt-smollm-32x1024", op="prompt", type="bf16", heads=9, kv=3, dim=64, seqs=32,
             least=64, most=1024, mix=10),
        # a 2048-token prefill (the prefill benchmark's largest) at BitNet-2B's shapes
        dict(name="prompt-bitnet-2048", op="prompt", type="f16", heads=20, kv=5, dim=128, seqs=1,
             least=2048, most=2048, mix=11),
        # two long documents in one call
        dict(name="prompt-long-2x8k", op="prompt", type="bf16", heads=20, kv=5, dim=128, seqs=2,
             least=6001, most=8192, mix=12),
    ]


def _spread(rng, lo, hi):
    """A whole number in [lo, hi], evenly spread over its logarithm."""
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["append", "append", "decode", "decode", "prompt", "prompt"])
    heads, kv, dim = rng.choice([(9, 3, 64), (20, 5, 128), (32, 8, 128), (32, 4, 128), (8, 8, 64),
                                 (12, 1, 128), (16, 2, 64), (5, 5, 128)])
    c = dict(op=op, type=rng.choice(["f32", "f16", "bf16"]), heads=heads, kv=kv, dim=dim,
             mix=rng.randrange(1 << 20))
    if op == "append":
        step = rng.random() < 0.5
        c |= dict(page=rng.choice([16, 32, 64, 128]), rot=rng.choice([dim, dim // 2, 16, dim - 8, 0]),
                  pairs=rng.choice([0, 1]), out=rng.choice(["f32", "f16", "bf16"]), copies=not step,
                  seqs=_spread(rng, 1, 100 if step else 24), least=1,
                  most=1 if step else _spread(rng, 2, 1500))
        if not step and rng.random() < 0.3:
            c["copies"] = False
    elif op == "decode":
        seqs = _spread(rng, 1, 256)
        c |= dict(page=rng.choice([16, 32, 64, 128]), seqs=seqs, out=c["type"],
                  most=_spread(rng, 1, min(100000, 1200000 // (seqs * kv))))
        c["least"] = rng.choice([0, 1, 1 + c["most"] // 2, c["most"]])
        c["least"] = min(c["least"], c["most"])
    else:
        seqs = _spread(rng, 1, 40)
        c |= dict(type=rng.choice(["f16", "bf16"]), seqs=seqs,
                  most=_spread(rng, 1, int((1e9 / (seqs * heads)) ** 0.5)))
        c["least"] = min(c["most"], rng.choice([1, 1 + c["most"] // 2, c["most"]]))
    return c


def lengths(case):
    """Tokens (append, prompt) or keys (decode) of each sequence: fixed by the case."""
    r = random.Random(case["mix"])
    n = [r.randint(case["least"], case["most"]) for _ in range(case["seqs"])]
    n[0] = case["most"]
    return n


def contexts(case):
    """append: tokens that each sequence has in the cache before the call (0: a new prompt).  A step's
    sequences stand anywhere in their last two pages; the pool holds no others, since an append
    neither reads nor writes them."""
    r = random.Random(case["mix"] + 1)
    if case["most"] == 1:
        return [r.randint(0, 2 * case["page"] - 1) for _ in range(case["seqs"])]
    return [r.choice([0, 0, r.randint(1, case["page"])]) for _ in range(case["seqs"])]


# ------------------------------------------------------------------------------------ inputs

def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _start(n):
    return torch.tensor(np.concatenate([[0], np.cumsum(n)]), dtype=torch.int32, device="cuda")


def _pages(case, g, tokens):
    """Page table and empty pool of a cache that holds `tokens` of each sequence, pages in random
    order; a few spare pages belong to nobody."""
    need = [-(-t // case["page"]) for t in tokens]
    most, total = max(1, max(need)), sum(need) + 3
    order = torch.randperm(total, generator=g, device="cuda").int()
    table = torch.zeros(len(need), most, dtype=torch.int32, device="cuda")
    used = torch.arange(most, device="cuda")[None, :] < torch.tensor(need, device="cuda")[:, None]
    table[used] = order[:sum(need)]
    shape = (total, case["kv"], case["page"], case["dim"])
    return {"table": table, "n_pages": total, "shape": shape}


def _codes(g, shape):
    """Codes as absmax quantisation of roughly normal rows leaves them, and a scale for each page and head."""
    q = torch.empty(shape, dtype=torch.int8, device="cuda")
    flat = q.view(-1)
    for i in range(0, flat.numel(), 1 << 26):
        n = min(1 << 26, flat.numel() - i)
        flat[i:i + n] = (torch.randn(n, generator=g, device="cuda") * 36).round_().clamp_(-127, 127).to(torch.int8)
    scale = (torch.rand(shape[:2], generator=g, device="cuda") * 0.03 + 0.015).contiguous()
    return q, scale


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 1000003 + case["mix"])
    H, KV, D, t = case["heads"], case["kv"], case["dim"], TYPES[case["type"]]
    n = lengths(case)
    s = {"case": case, "scale": D ** -0.5}
    if case["op"] == "append":
        T, before = sum(n), contexts(case)
        s |= _pages(case, g, [a + b for a, b in zip(n, before)])
        s["k_cache"], s["k_scale"] = _codes(g, s["shape"])
        s["v_cache"], s["v_scale"] = _codes(g, s["shape"])
        # one fused projection's output: q, k and v of a token side by side; a few channels of k are
        # larger than the rest, as trained models have them
        x = _normal(g, T, (H + 2 * KV) * D)
        x[:, H * D:(H + KV) * D:37] *= 4
        x = x.to(t)
        s["q"], s["k"], s["v"] = x[:, :H * D], x[:, H * D:(H + KV) * D], x[:, (H + KV) * D:]
        s["start"] = _start(n)
        s["position"] = torch.tensor(before, dtype=torch.int32, device="cuda")
        last = max(a + b for a, b in zip(n, before))
        freq = 10000.0 ** (-torch.arange(case["rot"] // 2, dtype=torch.float64, device="cuda") * 2 / max(1, case["rot"]))
        angle = torch.arange(last, dtype=torch.float64, device="cuda")[:, None] * freq
        s["rope"] = torch.stack([angle.cos(), angle.sin()], -1).float().contiguous()
        o = TYPES[case["out"]]
        s["q_out"] = torch.empty(T, H * D, dtype=o, device="cuda")
        if case["copies"]:
            s["k_out"] = torch.empty(T, KV * D, dtype=o, device="cuda")
            s["v_out"] = torch.empty(T, KV * D, dtype=o, device="cuda")
    elif case["op"] == "decode":
        s |= _pages(case, g, n)
        s["k_cache"], s["k_scale"] = _codes(g, s["shape"])
        s["v_cache"], s["v_scale"] = _codes(g, s["shape"])
        s["q"] = (_normal(g, case["seqs"], H * D) * 1.5).to(t)
        s["length"] = torch.tensor(n, dtype=torch.int32, device="cuda")
        s["out"] = torch.empty(case["seqs"], H * D, dtype=TYPES[case["out"]], device="cuda")
        # what wl_attn_decode_workspace_bytes asks for at most; zero before its first use
        s["workspace"] = torch.zeros(16 << 20, dtype=torch.uint8, device="cuda")
    else:
        T = sum(n)
        s["longest"] = max(n)
        s["start"] = _start(n)
        s["q"] = (_normal(g, T, H * D) * 1.5).to(t)
        s["k"], s["v"] = _normal(g, T, KV * D).to(t), _normal(g, T, KV * D).to(t)
        s["out"] = torch.empty(T, H * D, dtype=t, device="cuda")
    return s


# ------------------------------------------------------------------------------- plain forms

def _rotate(x, rope, pos, case):
    """x [T, heads, dim] f32, rotated in its first `rot` dimensions; products and sums rounded one by one."""
    rot = case["rot"]
    if not rot:
        return x
    cos, sin = rope[pos, :, 0][:, None, :], rope[pos, :, 1][:, None, :]
    head = x[..., :rot]
    a, b = (head[..., 0::2], head[..., 1::2]) if case["pairs"] else (head[..., :rot // 2], head[..., rot // 2:])
    u, w = a * cos - b * sin, a * sin + b * cos
    turned = torch.stack([u, w], -1).flatten(-2) if case["pairs"] else torch.cat([u, w], -1)
    return torch.cat([turned, x[..., rot:]], -1)


def _append_one(codes, scale, x, page, slot, first, fresh):
    """Appends x [T, kv, dim] f32 at (page, slot).  A page begun by this call takes absmax / 127 as its
    scale; one that was begun before keeps its scale, doubled as often as the new values need, and the
    codes in front of the new ones are rounded to the doubled steps."""
    need = torch.zeros_like(scale).scatter_reduce(0, page[:, None].expand(-1, x.shape[1]), x.abs().amax(-1), "amax")
    need = need / torch.full_like(need, 127)  # a quotient (by a plain number it is a product with 1 / 127)
    part, power = torch.frexp(need / scale)
    power = power - (part == 0.5).to(power.dtype)
    power = power + (torch.ldexp(scale, power) < need).to(power.dtype)  # the quotient was rounded
    grown = torch.where(need <= scale, scale, torch.where(scale == 0, need, torch.ldexp(scale, power)))
    new = torch.where(fresh[:, None], need, grown)
    halvings = torch.where(fresh[:, None] | (need <= scale) | (scale == 0), torch.zeros_like(power), power)
    old = torch.arange(codes.shape[2], device=x.device)[None, :] < first[:, None]
    moved = torch.round(torch.ldexp(codes.float(), -halvings[:, :, None, None])).to(torch.int8)
    codes.copy_(torch.where(old[:, None, :, None], moved, codes))
    scale.copy_(new)
    step = new[page][..., None]
    q = torch.where(step > 0, torch.round(x / step).clamp(-127, 127), torch.zeros_like(x))
    codes[page, :, slot] = q.to(torch.int8)


def _append(s):
    c, P = s["case"], s["case"]["page"]
    T = s["q"].shape[0]
    token = torch.arange(T, device="cuda")
    seq = torch.searchsorted(s["start"][1:], token.int(), right=True)
    pos = (s["position"][seq] + token - s["start"][seq]).long()
    page, slot = s["table"][seq, pos // P].long(), pos % P
    # the first slot that this call writes in each page (the page's size: none)
    first = torch.full((s["n_pages"],), P, device="cuda").scatter_reduce(0, page, slot, "amin")
    fresh = first == 0
    first = torch.where(first == P, torch.zeros_like(first), first)
    q, k, v = (s[n].float().view(T, -1, c["dim"]) for n in "qkv")
    q, k = _rotate(q, s["rope"], pos, c), _rotate(k, s["rope"], pos, c)
    _append_one(s["k_cache"], s["k_scale"], k, page, slot, first, fresh)
    _append_one(s["v_cache"], s["v_scale"], v, page, slot, first, fresh)
    s["q_out"].copy_(q.flatten(1))
    if c["copies"]:
        s["k_out"].copy_(k.flatten(1))
        s["v_out"].copy_(v.flatten(1))


def _decode(s):
    c = s["case"]
    S, G, D = c["seqs"], c["heads"] // c["kv"], c["dim"]
    table = s["table"].long()

    def rows(codes, scale):  # [seqs, kv, keys, dim]
        x = codes[table] * scale[table][..., None, None]
        return x.transpose(1, 2).reshape(S, c["kv"], -1, D)

    k = rows(s["k_cache"], s["k_scale"])
    q = s["q"].float().view(S, c["kv"], G, D) * s["scale"]
    score = q @ k.transpose(2, 3)
    del k
    here = torch.arange(score.shape[-1], device="cuda") < s["length"][:, None, None, None]
    score = score.masked_fill(~here, float("-inf"))
    top = score.amax(-1, keepdim=True).clamp_min(torch.finfo(torch.float32).min)
    p = torch.exp(score - top)
    total = p.sum(-1, keepdim=True)
    out = (p @ rows(s["v_cache"], s["v_scale"])) / torch.where(total > 0, total, torch.ones_like(total))
    s["out"].copy_(out.view(S, -1))


def _prompt(s):
    c, L = s["case"], s["longest"]
    S, H, KV, D = c["seqs"], c["heads"], c["kv"], c["dim"]
    start = s["start"].long()
    at = torch.arange(L, device="cuda")
    here = at[None, :] < (start[1:] - start[:-1])[:, None]
    rows = (start[:-1, None] + at).clamp_max(s["q"].shape[0] - 1)
    q = s["q"].float()[rows].view(S, L, KV, H // KV, D).permute(0, 2, 3, 1, 4) * s["scale"]
    k = s["k"].float()[rows].view(S, L, KV, 1, D).permute(0, 2, 3, 4, 1)
    v = s["v"].float()[rows].view(S, L, KV, 1, D).permute(0, 2, 3, 1, 4)
    p = (q.flatten(2, 3) @ k[:, :, 0]).view(S, KV, H // KV, L, L)
    p = p.masked_fill_(at[None, :] > at[:, None], float("-inf"))
    p = p.sub_(p.amax(-1, keepdim=True)).exp_()
    total = p.sum(-1, keepdim=True)
    out = (p.flatten(2, 3) @ v[:, :, 0]).view(S, KV, H // KV, L, D) / total
    s["out"].copy_(out.permute(0, 3, 1, 2, 4).reshape(S, L, H * D)[here])


# --------------------------------------------------------------------------- the library's calls

def _args(s):
    """The calls' argument structs: a program fills them once for its buffers."""
    from project_willamette_b200 import _abi
    c = s["case"]
    a = {"lib": _abi.lib()}
    if "k_cache" in s:
        a["cache"] = _abi.WlKvPagesI8(
            k=s["k_cache"].data_ptr(), v=s["v_cache"].data_ptr(), k_scale=s["k_scale"].data_ptr(),
            v_scale=s["v_scale"].data_ptr(), n_pages=s["n_pages"], page_size=c["page"],
            n_kv_heads=c["kv"], head_dim=c["dim"])
    if c["op"] == "append":
        a["call"] = _abi.WlKvAppend(
            q=s["q"].data_ptr(), k=s["k"].data_ptr(), v=s["v"].data_ptr(), q_stride=s["q"].stride(0),
            k_stride=s["k"].stride(0), v_stride=s["v"].stride(0), seq_start=s["start"].data_ptr(),
            position=s["position"].data_ptr(), page_table=s["table"].data_ptr(),
            rope=s["rope"].data_ptr() if c["rot"] else None, q_out=s["q_out"].data_ptr(),
            k_out=s["k_out"].data_ptr() if c["copies"] else None,
            v_out=s["v_out"].data_ptr() if c["copies"] else None, type=GGML[c["type"]],
            out_type=GGML[c["out"]], n_tokens=s["q"].shape[0], n_seqs=c["seqs"], n_q_heads=c["heads"],
            max_pages=s["table"].shape[1], n_rot=c["rot"], rope_len=s["rope"].shape[0],
            rope_pairs=c["pairs"])
    elif c["op"] == "decode":
        a["call"] = _abi.WlAttnDecode(
            q=s["q"].data_ptr(), out=s["out"].data_ptr(), q_stride=s["q"].stride(0),
            out_stride=s["out"].stride(0), length=s["length"].data_ptr(),
            page_table=s["table"].data_ptr(), workspace=s["workspace"].data_ptr(),
            workspace_bytes=s["workspace"].numel(), type=GGML[c["type"]],
            out_type=GGML[c["out"]], n_seqs=c["seqs"], n_q_heads=c["heads"],
            max_pages=s["table"].shape[1], scale=s["scale"])
    else:
        a["call"] = _abi.WlAttnPrompt(
            q=s["q"].data_ptr(), k=s["k"].data_ptr(), v=s["v"].data_ptr(), out=s["out"].data_ptr(),
            q_stride=s["q"].stride(0), k_stride=s["k"].stride(0), v_stride=s["v"].stride(0),
            out_stride=s["out"].stride(0), seq_start=s["start"].data_ptr(), type=GGML[c["type"]],
            out_type=GGML[c["type"]], n_tokens=s["q"].shape[0], n_seqs=c["seqs"],
            n_q_heads=c["heads"], n_kv_heads=c["kv"], head_dim=c["dim"], scale=s["scale"])
    return a


def _call(s):
    import ctypes as C
    a = s.get("args")
    if a is None:
        a = s["args"] = _args(s)
    L, stream, op = a["lib"], torch.cuda.current_stream().cuda_stream, s["case"]["op"]
    if op == "append":
        rc = L.wl_dev_rope_kv_append_i8(C.byref(a["cache"]), C.byref(a["call"]), stream)
    elif op == "decode":
        rc = L.wl_dev_attn_decode_i8(C.byref(a["cache"]), C.byref(a["call"]), stream)
    else:
        rc = L.wl_dev_attn_prompt(C.byref(a["call"]), stream)
    if rc:
        raise RuntimeError(L.wl_last_error().decode())


def run(state):
    op = state["case"]["op"]
    if own:
        _call(state)
    else:
        {"append": _append, "decode": _decode, "prompt": _prompt}[op](state)
    if op != "append":
        return {"out": state["out"]}
    r = {n: state[n] for n in ("q_out", "k_out", "v_out") if n in state}
    for n in "kv":  # the cache as the values that its codes stand for
        r[n + "_cache"] = state[n + "_cache"] * state[n + "_scale"][..., None, None]
    return r


# ------------------------------------------------------------------------------------- work

def work(case):
    H, KV, D, n = case["heads"], case["kv"], case["dim"], lengths(case)
    size = {"f32": 4, "f16": 2, "bf16": 2}
    T = sum(n)
    if case["op"] == "append":
        codes, before = 0, contexts(case)
        for a, b in zip(before, n):  # codes written; a page that was begun before is read too when its scale grows
            codes += 2 * KV * D * b
        b = T * (H + 2 * KV) * D * size[case["type"]] + codes
        b += T * (H + (2 * KV if case["copies"] else 0)) * D * size[case["out"]]
        b += len(set(x for a, m in zip(before, n) for x in range(a, a + m))) * case["rot"] * 4
        return {"bytes": b, "flops": 3 * T * (H + KV) * case["rot"]}
    if case["op"] == "decode":
        b = 2 * T * KV * D + 2 * sum(-(-x // case["page"]) for x in n) * KV * 4
        b += case["seqs"] * H * D * (size[case["type"]] + size[case["out"]])
        return {"bytes": b, "flops": 4 * T * H * D}
    pairs = sum(x * (x + 1) // 2 for x in n)
    return {"bytes": 2 * T * (H + KV) * D * size[case["type"]], "flops": 4 * pairs * H * D}


# ------------------------------------------------------------------------------------ exact

def _exact_append(s):
    """The operator's definition, sequence by sequence: its roundings to 32 bits (rotated values, scales
    and quotients, which the codes are rounded from) are made one at a time from 64-bit values."""
    c, P = s["case"], s["case"]["page"]
    D, rot = c["dim"], c["rot"]
    r32 = lambda x: x.float().double()  # noqa: E731
    n, before = lengths(c), contexts(c)
    table = s["table"].cpu().tolist()
    rope = s["rope"].double()
    x = {k: s[k].double().view(s[k].shape[0], -1, D).clone() for k in "qkv"}
    codes = {k: s[k + "_cache"].double() for k in "kv"}
    scale = {k: s[k + "_scale"].double() for k in "kv"}
    pos = torch.cat([torch.arange(b, b + m, device="cuda") for m, b in zip(n, before)])
    if rot:
        i = torch.arange(rot // 2, device="cuda")
        lo, hi = (2 * i, 2 * i + 1) if c["pairs"] else (i, i + rot // 2)
        co, si = rope[pos][:, None, :, 0], rope[pos][:, None, :, 1]
        for k in "qk":
            a, b = x[k][:, :, lo], x[k][:, :, hi]
            x[k][:, :, lo] = r32(r32(a * co) - r32(b * si))
            x[k][:, :, hi] = r32(r32(a * si) + r32(b * co))
    at = 0
    for q, (m, b) in enumerate(zip(n, before)):
        for j in range(b // P, -(-(b + m) // P)):
            lo, hi = max(b, j * P), min(b + m, (j + 1) * P)
            page = table[q][j]
            for k in "kv":
                new = x[k][at + lo - b:at + hi - b]  # [rows, kv, dim]
                need = r32(new.abs().amax((0, 2)) / 127)
                old, first = scale[k][page], lo - j * P
                if first == 0:
                    step = need
                else:
                    halvings = torch.zeros_like(old)
                    step = old.clone()
                    for _ in range(300):  # as often as needed, no more
                        short = (old > 0) & (need > step)
                        step = torch.where(short, step * 2, step)
                        halvings += short
                    step = torch.where(old == 0, need, step)
                    codes[k][page, :, :first] = torch.round(codes[k][page, :, :first] / (2 ** halvings)[:, None, None])
                scale[k][page] = step
                w = step[None, :, None]
                codes[k][page, :, first:first + hi - lo] = torch.where(
                    w > 0, torch.round(r32(new / w)).clamp(-127, 127), torch.zeros_like(new)).transpose(0, 1)
        at += m
    r = {"q_out": x["q"].flatten(1)}
    if c["copies"]:
        r |= {"k_out": x["k"].flatten(1), "v_out": x["v"].flatten(1)}
    return r | {k + "_cache": codes[k] * scale[k][..., None, None] for k in "kv"}


def _softmax_rows(score, v):
    e = torch.exp(score - score.max(-1, keepdim=True).values)
    return torch.matmul(e / e.sum(-1, keepdim=True), v)


def _exact_decode(s):
    c, n = s["case"], lengths(s["case"])
    out = torch.zeros(c["seqs"], c["heads"], c["dim"], dtype=torch.float64, device="cuda")
    G = c["heads"] // c["kv"]
    for i, m in enumerate(n):
        if not m:
            continue
        pages = s["table"][i, :-(-m // c["page"])].long()
        for h in range(c["kv"]):
            k, v = ((s[x + "_cache"][pages, h].double() * s[x + "_scale"][pages, h].double()[:, None, None])
                    .reshape(-1, c["dim"])[:m] for x in "kv")
            q = s["q"][i].double().view(-1, c["dim"])[h * G:(h + 1) * G]
            out[i, h * G:(h + 1) * G] = _softmax_rows(torch.matmul(q, k.T) * s["scale"], v)
    return {"out": out.flatten(1)}


def _exact_prompt(s):
    c, n = s["case"], lengths(s["case"])
    D, G = c["dim"], c["heads"] // c["kv"]
    q, k, v = (s[x].double().view(s[x].shape[0], -1, D) for x in "qkv")
    out = torch.empty_like(q)
    at = 0
    for m in n:
        above = torch.ones(m, m, dtype=torch.bool, device="cuda").triu(1)
        for h in range(c["heads"]):
            score = torch.matmul(q[at:at + m, h], k[at:at + m, h // G].T) * s["scale"]
            out[at:at + m, h] = _softmax_rows(score.masked_fill(above, -torch.inf), v[at:at + m, h // G])
        at += m
    return {"out": out.flatten(1)}


def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "decode": _exact_decode, "prompt": _exact_prompt}[case["op"]](s)
