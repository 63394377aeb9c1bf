"""Plain implementations of the paged int8 cache operators for their tests, and
the calls as small functions over torch tensors."""
import ctypes as C

import numpy as np
import torch

from project_willamette_b200 import _abi

GGML = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 30}


def half_step(dtype):
    """Half a rounding step, relative to the value."""
    return torch.finfo(dtype).eps / 2


def ptr(t):
    return None if t is None else t.data_ptr()


class Cache:
    """A paged cache with its page tables on `device`."""

    def __init__(self, n_pages, page, kv, dim, device="cuda", fill=0):
        shape = (n_pages, kv, page, dim)
        self.k = torch.full(shape, fill, dtype=torch.int8, device=device)
        self.v = torch.full(shape, fill, dtype=torch.int8, device=device)
        self.ks = torch.zeros(n_pages, kv, device=device)
        self.vs = torch.zeros(n_pages, kv, device=device)
        self.page, self.kv, self.dim = page, kv, dim

    def struct(self, **other):
        return _abi.WlKvPagesI8(**{**dict(
            k=ptr(self.k), v=ptr(self.v), k_scale=ptr(self.ks), v_scale=ptr(self.vs),
            n_pages=self.k.shape[0], page_size=self.page, n_kv_heads=self.kv, head_dim=self.dim),
            **other})

    def clone(self):
        c = object.__new__(Cache)
        c.__dict__ = {n: x.clone() if torch.is_tensor(x) else x for n, x in self.__dict__.items()}
        return c


def i32(values, device="cuda"):
    return torch.tensor(values, dtype=torch.int32, device=device)


def starts(lengths, device="cuda"):
    return i32(np.concatenate([[0], np.cumsum(lengths)]).tolist(), device)


def rope_table(length, n_rot, base=10000.0, factor=1.0):
    """(cos, sin) rows, angles in 64 bits; `factor` > 1 stretches positions for a longer context."""
    f = base ** (-np.arange(n_rot // 2, dtype=np.float64) * 2 / max(n_rot, 1))
    a = np.arange(length, dtype=np.float64)[:, None] / factor * f
    return np.stack([np.cos(a), np.sin(a)], -1).astype(np.float32)


def append_args(q, k, v, start, position, table, rope, n_rot, pairs, out_type, q_out=None, k_out=None,
                v_out=None, heads=0, n_tokens=None, **other):
    a = dict(q=ptr(q), k=ptr(k), v=ptr(v), q_stride=q.stride(0) if q is not None else 0,
             k_stride=k.stride(0), v_stride=v.stride(0), seq_start=ptr(start), position=ptr(position),
             page_table=ptr(table), rope=ptr(rope), q_out=ptr(q_out), k_out=ptr(k_out),
             v_out=ptr(v_out), type=GGML[k.dtype], out_type=GGML[out_type],
             n_tokens=k.shape[0] if n_tokens is None else n_tokens, n_seqs=position.numel(),
             n_q_heads=heads, max_pages=table.shape[1], n_rot=n_rot,
             rope_len=rope.shape[0] if rope is not None else 0, rope_pairs=pairs)
    return _abi.WlKvAppend(**{**a, **other})


def stream():
    return torch.cuda.current_stream().cuda_stream


def check(rc):
    assert rc == 0, _abi.lib().wl_last_error()


def append(cache, args):
    check(_abi.lib().wl_dev_rope_kv_append_i8(C.byref(cache.struct()), C.byref(args), stream()))


def workspace(seqs, heads, cache):
    n = _abi.lib().wl_attn_decode_workspace_bytes(seqs, heads, cache.kv, cache.dim)
    return torch.zeros(n, dtype=torch.uint8, device="cuda")


def decode_args(q, out, length, table, ws, scale, **other):
    a = dict(q=ptr(q), out=ptr(out), q_stride=q.stride(0), out_stride=out.stride(0),
             length=ptr(length), page_table=ptr(table), workspace=ptr(ws), workspace_bytes=ws.numel(),
             type=GGML[q.dtype], out_type=GGML[out.dtype], n_seqs=q.shape[0],
             n_q_heads=other.pop("heads"), max_pages=table.shape[1], scale=scale)
    return _abi.WlAttnDecode(**{**a, **other})


def decode(cache, q, length, table, heads, scale, ws=None, out=None, out_type=None):
    ws = workspace(q.shape[0], heads, cache) if ws is None else ws
    if out is None:
        out = torch.full((q.shape[0], heads * cache.dim), float("nan"), dtype=out_type or q.dtype,
                         device="cuda")
    a = decode_args(q, out, length, table, ws, scale, heads=heads)
    check(_abi.lib().wl_dev_attn_decode_i8(C.byref(cache.struct()), C.byref(a), stream()))
    return out


def prompt_args(q, k, v, out, start, heads, kv, dim, scale, **other):
    a = dict(q=ptr(q), k=ptr(k), v=ptr(v), out=ptr(out), q_stride=q.stride(0), k_stride=k.stride(0),
             v_stride=v.stride(0), out_stride=out.stride(0), seq_start=ptr(start), type=GGML[q.dtype],
             out_type=GGML[out.dtype], n_tokens=q.shape[0], n_seqs=start.numel() - 1,
             n_q_heads=heads, n_kv_heads=kv, head_dim=dim, scale=scale)
    return _abi.WlAttnPrompt(**{**a, **other})


def prompt(q, k, v, start, heads, kv, dim, scale, out=None, out_type=None):
    if out is None:
        out = torch.full((q.shape[0], heads * dim), float("nan"), dtype=out_type or q.dtype,
                         device="cuda")
    a = prompt_args(q, k, v, out, start, heads, kv, dim, scale)
    check(_abi.lib().wl_dev_attn_prompt(C.byref(a), stream()))
    return out


def status():
    w = C.c_uint32(0xFFFFFFFF)
    check(_abi.lib().wl_device_status(C.byref(w)))
    return w.value


# ------------------------------------------------------------------ the definitions, on the host

def rotate(x, rope, pos, n_rot, pairs):
    """x [rows, heads, dim] f32 (numpy), each product and sum rounded to f32."""
    x = x.copy()
    if not n_rot:
        return x
    i = np.arange(n_rot // 2)
    lo, hi = (2 * i, 2 * i + 1) if pairs else (i, i + n_rot // 2)
    c, s = rope[pos][:, None, :, 0], rope[pos][:, None, :, 1]
    a, b = x[..., lo], x[..., hi]
    x[..., lo] = a * c - b * s
    x[..., hi] = a * s + b * c
    return x


def append_rows(codes, scale, page, first, rows):
    """rows [n, kv, dim] f32 into `page` from row `first` on; codes and scale are numpy arrays."""
    f32 = np.float32
    for h in range(rows.shape[1]):
        x = rows[:, h]
        need = np.abs(x).max() / f32(127) if np.isfinite(x).all() else f32(np.nan)
        old = scale[page, h]
        if first == 0 or np.isnan(need):
            s = need
        elif np.isnan(old) or need <= old:
            s = old
        elif old == 0:
            s = need
        else:
            s, k = old, 0
            while s < need:
                s, k = f32(s * f32(2)), k + 1
            codes[page, h, :first] = np.rint(np.ldexp(codes[page, h, :first].astype(np.float64), -k))
        scale[page, h] = s
        q = np.clip(np.rint(x / s), -127, 127) if s > 0 else np.zeros_like(x)
        codes[page, h, first:first + len(x)] = q


def append_ref(cache, q, k, v, lengths, position, table, rope, n_rot, pairs):
    """The cache after the call (numpy: k, ks, v, vs) and the rotated q and k, v (f32)."""
    D, P = cache.dim, cache.page
    c = [cache.k.cpu().numpy().copy(), cache.ks.cpu().numpy().copy(),
         cache.v.cpu().numpy().copy(), cache.vs.cpu().numpy().copy()]
    f = [None if t is None else t.float().cpu().numpy().reshape(t.shape[0], -1, D) for t in (q, k, v)]
    pos = np.concatenate([np.arange(b, b + n) for n, b in zip(lengths, position)]).astype(np.int64)
    T = len(pos)
    f = [None if x is None else x[:T] for x in f]
    with np.errstate(all="ignore"):
        rq = None if q is None else rotate(f[0], rope, pos, n_rot, pairs)
        rk = rotate(f[1], rope, pos, n_rot, pairs)
        at = 0
        for s, (n, b) in enumerate(zip(lengths, position)):
            for j in range(b // P, -(-(b + n) // P) if n else 0):
                lo, hi = max(b, j * P), min(b + n, (j + 1) * P)
                for x, i in ((rk, 0), (f[2], 2)):
                    append_rows(c[i], c[i + 1], int(table[s][j]), lo - j * P,
                                x[at + lo - b:at + hi - b])
            at += n
    return c, rq, rk, f[2]


def softmax_rows(z, v):
    """(softmax(z) v, softmax(z) |v|) in 64 bits; z [.., rows, keys]."""
    e = torch.exp(z - z.amax(-1, keepdim=True))
    w = e / e.sum(-1, keepdim=True)
    return w @ v, w @ v.abs()


def decode_ref(cache, q, length, table, heads, scale):
    """out and its allowance, both [seqs, heads * dim] in 64 bits.

    What the f32 path may be off by, with w the softmax weights: each weight by the error of its
    exponent, twice (once in the sum below the line): the dot product's dim + 4 roundings of
    2^-24, relative to scale * |q| . |k| (a split of q in two 16-bit parts has 22 bits and counts as
    four more), plus 2^-20 for exp, exponent and scale products; the sums over keys by one
    rounding per key.  A weight also has an absolute error: as e^(z - m) * 2^14, at most 2^14, it is
    split into two f16 numbers whose remainder is at most half of f16's smallest, 2^-25, so 2^-39
    of the largest weight, which is 1 before the division by a sum of at least 1; it multiplies
    |code| and, since weights are taken relative to it, the largest scale."""
    S, G, D = q.shape[0], heads // cache.kv, cache.dim
    out = torch.zeros(S, heads, D, dtype=torch.float64, device="cuda")
    tol = torch.zeros_like(out)
    for i in range(S):
        n = int(length[i])
        if not n:
            continue
        pages = table[i, :-(-n // cache.page)].long()
        for h in range(cache.kv):
            k = (cache.k[pages, h].double() * cache.ks[pages, h].double()[:, None, None]).reshape(-1, D)[:n]
            v = (cache.v[pages, h].double() * cache.vs[pages, h].double()[:, None, None]).reshape(-1, D)[:n]
            x = q[i].double().view(-1, D)[h * G:(h + 1) * G]
            z = x @ k.T * scale
            size = (x.abs() @ k.abs().T * abs(scale)).amax(-1, keepdim=True)
            out[i, h * G:(h + 1) * G], a = softmax_rows(z, v)
            tol[i, h * G:(h + 1) * G] = a * (2 * (size * (D + 8) * 2.0 ** -24 + 2.0 ** -20) + (n + 64) * 2.0 ** -24)
            c_abs = cache.v[pages, h].double().abs().reshape(-1, D)[:n].sum(0)
            tol[i, h * G:(h + 1) * G] += 2.0 ** -39 * cache.vs[pages, h].double().max() * c_abs
    return out.flatten(1), tol.flatten(1)


def prompt_ref(q, k, v, lengths, heads, kv, dim, scale):
    """out and its allowance for the rows that sequences own: as decode_ref, and each weight's
    rounding to the inputs' 16-bit type."""
    G = heads // kv
    T = sum(lengths)
    a, b, c = (x[:T].double().view(T, -1, dim) for x in (q, k, v))
    out = torch.empty(T, heads, dim, dtype=torch.float64, device="cuda")
    tol = torch.empty_like(out)
    at = 0
    for n in lengths:
        above = torch.ones(n, n, dtype=torch.bool, device="cuda").triu(1)
        for h in range(heads if n else 0):
            x, y, w = a[at:at + n, h], b[at:at + n, h // G], c[at:at + n, h // G]
            z = (x @ y.T * scale).masked_fill(above, -torch.inf)
            size = (x.abs() @ y.abs().T * abs(scale)).masked_fill(above, 0).amax(-1, keepdim=True)
            o, m = softmax_rows(z, w)
            out[at:at + n, h] = o
            tol[at:at + n, h] = m * (2 * (size * (dim + 8) * 2.0 ** -24 + 2.0 ** -20) +
                                     (n + 64) * 2.0 ** -24 + half_step(q.dtype))
        at += n
    return out.flatten(1), tol.flatten(1)


def within(got, ref, tol):
    """got is ref, off by at most tol and one rounding to got's type."""
    g = got.double()
    assert torch.isfinite(g).all()
    far = (g - ref).abs() - (tol * 1.001 + ref.abs() * half_step(got.dtype) * 1.001 + tol * half_step(got.dtype))
    # below the type's normal range a rounding is half a step of the smallest number
    far = far - torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps / 2
    assert (far <= 0).all(), float(far.max())
