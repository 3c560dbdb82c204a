"""Rotary positions, the 8-bit KV cache's write and read, and the decode
attention over it: the calls that are timed, with a plain torch form of each.

Three operators, one attention layer of a decode step between them:

  rope       optional per-head RMSNorm, then the rotary rotation of the first
             rot dims of every q and k head (half or interleaved pairs), with
             plain, linear, NTK or YaRN frequencies
  kv8_write  K and V rows into the paged 8-bit cache (blocks of 16 tokens of
             one head share a power-of-two scale), and the touched blocks read
             back as the values the codes stand for
  kv8_attn   one query token per sequence over the cached tokens, with the
             layer's sigmoid output gate or without

`own` false: the plain forms.  `own` true: include/qrope.h and
include/qkv8.h, through the package's qcache module.
"""
import importlib.util
import math
import os
import sys

import numpy as np
import torch

own = False

PAGE, BLOCK = 64, 16
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
EPS = 1e-6


def _qcache():
    full = "qcache_b200_qcache"
    if full not in sys.modules:
        path = os.path.join(ROOT, "qwen3.5-9b-bfp8b-1xn300_b200", "qcache.py")
        spec = importlib.util.spec_from_file_location(full, path)
        sys.modules[full] = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(sys.modules[full])
    return sys.modules[full]


def _stream():
    return torch.cuda.current_stream().cuda_stream


# ------------------------------------------------------------------- cases

def listed():
    return [
        # the model's heads (16 query, 4 kv of 256; 64 dims rotate), taken from projection rows
        # [16][q | gate], k, v: one decode step of 8 sequences
        dict(name="rope_decode_8", op="rope", rows=8, nq=16, nk=4, dim=256, rot=64, half=True, norm=True,
             fused=True, scaling="plain", base=1e7, factor=1.0, orig=0, far=131072),
        # a 2048-token prompt of the same model beyond its trained context
        dict(name="rope_prompt_2048_yarn", op="rope", rows=2048, nq=16, nk=4, dim=256, rot=64, half=True, norm=True,
             fused=True, scaling="yarn", base=1e7, factor=4.0, orig=131072, far=524288),
        # a large prefill batch with 128-wide heads rotated whole in interleaved pairs
        dict(name="rope_interleaved_32768", op="rope", rows=32768, nq=32, nk=8, dim=128, rot=128, half=False,
             norm=False, fused=False, scaling="linear", base=1e4, factor=8.0, orig=8192, far=32768),
        # one new token for each of 64 sequences, most of them inside a block
        dict(name="write_step_64", op="write", n=64, lo=1, hi=1, kv=4, dim=256, ctx=4096, fused=True),
        # a 2048-token prompt moved into the cache
        dict(name="write_prompt_2048", op="write", n=1, lo=2048, hi=2048, kv=4, dim=256, ctx=0, fused=False),
        # prompt chunks of 16 sequences, odd starts and lengths
        dict(name="write_ragged_16", op="write", n=16, lo=1, hi=3999, kv=4, dim=256, ctx=2000, fused=False),
        # a 65536-token history converted at once, 8 heads of 128
        dict(name="write_history_65536", op="write", n=1, lo=65536, hi=65536, kv=8, dim=128, ctx=0, fused=False),
        # one sequence at 1024 tokens: latency
        dict(name="attn_1x1024", op="attn", n=1, lo=1024, hi=1024, kv=4, group=4, dim=256, gate=True),
        # the headline batch: 64 sequences of 4096
        dict(name="attn_64x4096", op="attn", n=64, lo=4096, hi=4096, kv=4, group=4, dim=256, gate=True),
        # one long context
        dict(name="attn_1x131072", op="attn", n=1, lo=131072, hi=131072, kv=4, group=4, dim=256, gate=True),
        # a ragged batch, one slot of it empty, 6 query heads to a kv head of 128
        dict(name="attn_ragged_33", op="attn", n=33, lo=0, hi=8191, kv=2, group=6, dim=128, gate=False),
        # a small batch of short contexts, 64-wide heads, 8 to a kv head
        dict(name="attn_9x300", op="attn", n=9, lo=1, hi=300, kv=1, group=8, dim=64, gate=False),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rope", "write", "attn", "attn"])
    if op == "rope":
        dim = rng.choice([64, 128, 256])
        rot = rng.choice([r for r in (16, 24, 32, 64, 96, 128, 256) if r <= dim])
        nq, nk = rng.choice([(16, 4), (32, 8), (24, 8), (8, 1), (20, 5)])
        most = 335_000_000 // (2 * dim * (nq + nk))
        scaling = rng.choice(["plain", "linear", "ntk", "yarn"])
        return dict(op="rope", rows=_log_int(rng, 1, min(32768, most)), nq=nq, nk=nk, dim=dim, rot=rot,
                    half=rng.random() < 0.6, norm=rng.random() < 0.5, fused=rng.random() < 0.5, scaling=scaling,
                    base=rng.choice([1e4, 5e5, 1e7]), factor=1.0 if scaling == "plain" else rng.choice([2.0, 4.0, 8.0]),
                    orig=rng.choice([8192, 32768, 131072]), far=_log_int(rng, 64, 1 << 20))
    dim = rng.choice([64, 128, 256])
    kv = rng.choice([1, 2, 3, 4, 8])
    if op == "write":
        n = _log_int(rng, 1, 128)
        hi = _log_int(rng, 1, max(1, min(32768, 65536 * 1024 // (n * kv * dim))))
        return dict(op="write", n=n, lo=rng.choice([0, 1, hi]), hi=hi, kv=kv, dim=dim, ctx=rng.choice([0, 100, 5000]),
                    fused=rng.random() < 0.5)
    n = _log_int(rng, 1, 128)
    hi = _log_int(rng, 1, max(16, min(131072, 64 * 4096 * 1024 // (n * kv * dim))))
    return dict(op="attn", n=n, lo=rng.choice([0, hi // 2, hi]), hi=hi, kv=kv, group=rng.choice([1, 2, 4, 5, 6, 8]),
                dim=dim, gate=rng.random() < 0.5)


# ------------------------------------------------------------------ inputs

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(g, *shape, std=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(torch.bfloat16)


def _lengths(case):
    """Tokens of each sequence: the ends of the range, the rest uniform between them; the same whatever the seed."""
    r = np.random.default_rng([case["n"], case["lo"], case["hi"]])
    x = r.integers(case["lo"], case["hi"] + 1, case["n"])
    x[-1], x[0] = case["lo"], case["hi"]
    return x.astype(np.int64)


def _starts(case):
    """Tokens that each sequence of a write has already."""
    return np.random.default_rng(case["n"] + case["ctx"]).integers(0, case["ctx"] + 1, case["n"])


def _i32(x):
    return torch.from_numpy(np.ascontiguousarray(x, np.int32)).cuda()


def _table(lens, seed):
    """A page table of permuted pages for these lengths, and the number of pages in the pool."""
    per = np.maximum(1, -(-lens // PAGE))
    total, width = int(per.sum()), int(per.max())
    ids = np.random.default_rng(seed + 1).permutation(total + 3)[:total]
    t = np.zeros((len(lens), width), np.int32)
    t[np.arange(width)[None] < per[:, None]] = ids
    return _i32(t), total + 3


def _channels(g, kv, dim):
    """Standard deviations of K's channels: a few of them several times the rest, as keys have them."""
    s = torch.exp(0.5 * torch.randn(kv, dim, generator=g, device="cuda"))
    return s / s.square().mean(-1, keepdim=True).sqrt()


def _inputs(case, seed):
    g, s = _gen(seed), {}
    if case["op"] == "rope":
        rows, nq, nk, dim = case["rows"], case["nq"], case["nk"], case["dim"]
        if case["fused"]:   # one projection row: [nq][q | gate], k, v
            proj = _normal(g, rows, 2 * nq * dim + 2 * nk * dim)
            q = proj[:, :2 * nq * dim].unflatten(1, (nq, 2 * dim))[:, :, :dim]
            k = proj[:, 2 * nq * dim:2 * nq * dim + nk * dim].unflatten(1, (nk, dim))
        else:
            q, k = _normal(g, rows, nq, dim), _normal(g, rows, nk, dim)
        s.update(q=q, k=k, pos=torch.randint(0, case["far"], (rows,), generator=g, device="cuda", dtype=torch.int32))
        if case["norm"]:
            s["qw"] = 1 + 0.02 * torch.randn(dim, generator=g, device="cuda")
            s["kw"] = 1 + 0.02 * torch.randn(dim, generator=g, device="cuda")
    elif case["op"] == "write":
        n, kv, dim = case["n"], case["kv"], case["dim"]
        cnt, pos = _lengths(case), _starts(case)
        keep = pos % BLOCK              # older tokens in the block that the new ones go on in
        rows, std = int(cnt.sum()), _channels(g, kv, dim)
        if case["fused"]:               # k and v side by side in one row, as a projection gives them
            kvrow = torch.stack([torch.randn(rows, kv, dim, generator=g, device="cuda") * std,
                                 torch.randn(rows, kv, dim, generator=g, device="cuda")], 1).to(torch.bfloat16)
            k, v = kvrow[:, 0], kvrow[:, 1]
        else:
            k = (torch.randn(rows, kv, dim, generator=g, device="cuda") * std).to(torch.bfloat16)
            v = _normal(g, rows, kv, dim)
        old = int(keep.sum())
        s.update(k=k, v=v, n=n, rows=rows,
                 old_k=(torch.randn(old, kv, dim, generator=g, device="cuda") * std * 0.7).to(torch.bfloat16),
                 old_v=_normal(g, old, kv, dim, std=0.7),
                 pos=_i32(pos), start=_i32(np.concatenate([[0], np.cumsum(cnt)])),
                 old_pos=_i32(pos - keep), old_start=_i32(np.concatenate([[0], np.cumsum(keep)])), old_rows=old,
                 back_start=_i32(np.concatenate([[0], np.cumsum(cnt + keep)])), back_rows=rows + old)
        s["table"], s["pages"] = _table(pos + cnt, seed)
    else:
        n, kv, dim, heads = case["n"], case["kv"], case["dim"], case["kv"] * case["group"]
        lens = _lengths(case)
        rows = int(lens.sum())
        std = _channels(g, kv, dim)
        s.update(k=(torch.randn(rows, kv, dim, generator=g, device="cuda") * std).to(torch.bfloat16),
                 v=_normal(g, rows, kv, dim), n=n, rows=rows, heads=heads, pos=_i32(np.zeros(n)),
                 start=_i32(np.concatenate([[0], np.cumsum(lens)])), len=_i32(lens), scale=dim ** -0.5)
        qg = _normal(g, n, heads, 2 * dim, std=1.5)     # [heads][q | gate], as in a projection row
        s["q"], s["gate"] = (qg[:, :, :dim], qg[:, :, dim:]) if case["gate"] else (qg[:, :, :dim].contiguous(), None)
        s["table"], s["pages"] = _table(lens, seed)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    op, dim = case["op"], case["dim"]
    if op == "rope":
        if own:     # the frequencies are a user's constants, the outputs a user's buffers
            qc = _qcache()
            s["rope"] = qc.Rope(case["rot"], layout=qc.ROPE_HALF if case["half"] else qc.ROPE_INTERLEAVED,
                                base=case["base"], scaling=_kind(qc, case["scaling"]), factor=case["factor"],
                                orig_ctx=case["orig"])
            s["qo"], s["ko"] = torch.empty(s["q"].shape, dtype=torch.bfloat16, device="cuda"), torch.empty(
                s["k"].shape, dtype=torch.bfloat16, device="cuda")
        return s
    # the cache as the sequence's earlier tokens left it: for a write the tokens of the block that it goes on in, for
    # the attention all of them.  A program holds it in the form that its own calls keep it in.
    pos, start, rows, k, v = ("old_pos", "old_start", "old_rows", "old_k", "old_v") if op == "write" else (
        "pos", "start", "rows", "k", "v")
    if own:
        qc = _qcache()
        s["pool"] = torch.zeros(s["pages"] * qc.kv8_page_bytes(case["kv"], dim), dtype=torch.uint8, device="cuda")
        s["cache"] = qc.Kv8Cache(s["pool"].data_ptr(), s["pages"], case["kv"], dim)
        if s[rows]:
            s["cache"].write(s["table"].data_ptr(), s["table"].shape[1], s[pos].data_ptr(), s[start].data_ptr(), s["n"],
                             s[rows], s[k].data_ptr(), s[k].stride(0), s[v].data_ptr(), s[v].stride(0), _stream())
    else:
        s["codes"] = torch.zeros(2, s["pages"] * 4, BLOCK, case["kv"], dim, dtype=torch.int8, device="cuda")
        s["scales"] = torch.full((2, s["pages"] * 4, case["kv"]), 2.0 ** -126, device="cuda")
        if s[rows]:
            _plain_write(s, s[k], s[v], s[pos], s[start], s[rows])
    if op == "write":
        shape = (s["back_rows"], case["kv"], dim)
        s["kb"], s["vb"] = (torch.empty(shape, dtype=torch.bfloat16, device="cuda") for _ in "kv")
    else:
        s["out"] = torch.empty(s["n"], s["heads"], dim, dtype=torch.bfloat16, device="cuda")
        if own:
            need = s["cache"].attn_workspace_bytes(s["n"], s["heads"])
            s["work"] = torch.empty(max(1, need), dtype=torch.uint8, device="cuda")
        else:
            del s["k"], s["v"]
    return s


def _kind(qc, scaling):
    return dict(plain=qc.ROPE_PLAIN, linear=qc.ROPE_LINEAR, ntk=qc.ROPE_NTK, yarn=qc.ROPE_YARN)[scaling]


# --------------------------------------------------------------- one pass

def run(s):
    op = s["case"]["op"]
    if own:
        return _own_rope(s) if op == "rope" else _own_write(s) if op == "write" else _own_attn(s)
    if op == "rope":
        return [_plain_rope(s["case"], s["q"], s["pos"], s.get("qw")), _plain_rope(s["case"], s["k"], s["pos"], s.get("kw"))]
    if op == "write":
        _plain_write(s, s["k"], s["v"], s["pos"], s["start"], s["rows"])
        return _plain_read(s, s["old_pos"], s["back_start"], s["back_rows"])
    return _plain_attn(s)


def _own_rope(s):
    qc, case = _qcache(), s["case"]
    q, k, qo, ko = s["q"], s["k"], s["qo"], s["ko"]
    parts = [qc.RopePart(q.data_ptr(), qo.data_ptr(), case["nq"], q.stride(0), q.stride(1), qo.stride(0), qo.stride(1),
                         s["qw"].data_ptr() if case["norm"] else 0),
             qc.RopePart(k.data_ptr(), ko.data_ptr(), case["nk"], k.stride(0), k.stride(1), ko.stride(0), ko.stride(1),
                         s["kw"].data_ptr() if case["norm"] else 0)]
    s["rope"].apply(case["dim"], s["pos"].data_ptr(), case["rows"], parts, EPS, _stream())
    return [qo, ko]


def _own_write(s):
    c, t, st = s["cache"], s["table"], _stream()
    c.write(t.data_ptr(), t.shape[1], s["pos"].data_ptr(), s["start"].data_ptr(), s["n"], s["rows"], s["k"].data_ptr(),
            s["k"].stride(0), s["v"].data_ptr(), s["v"].stride(0), st)
    c.read(t.data_ptr(), t.shape[1], s["old_pos"].data_ptr(), s["back_start"].data_ptr(), s["n"], s["back_rows"],
           s["kb"].data_ptr(), s["kb"].stride(0), s["vb"].data_ptr(), s["vb"].stride(0), st)
    return [s["kb"], s["vb"]]


def _own_attn(s):
    t, q, g, out = s["table"], s["q"], s["gate"], s["out"]
    s["cache"].attn_decode(t.data_ptr(), t.shape[1], s["len"].data_ptr(), s["n"], s["heads"], q.data_ptr(), q.stride(0),
                           q.stride(1), g.data_ptr() if g is not None else 0, s["scale"], out.data_ptr(), out.stride(0),
                           s["work"].data_ptr(), s["work"].numel(), _stream())
    return [out]


# ------------------------------------------------------------ plain forms

def _frequencies(case):
    """Angle per position of each pair (64 bits), and the factor on the rotated values."""
    rot, base, f = case["rot"], case["base"], case["factor"]
    i = torch.arange(rot // 2, dtype=torch.float64, device="cuda")
    if case["scaling"] == "ntk":
        base = base * f ** (rot / (rot - 2))
    w = base ** (-2 * i / rot)
    if case["scaling"] == "linear":
        return w / f, 1.0
    if case["scaling"] != "yarn":
        return w, 1.0
    turn = lambda b: rot * math.log(case["orig"] / (b * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
    low, high = max(math.floor(turn(32.0)), 0), min(math.ceil(turn(1.0)), rot - 1)
    ramp = ((i - low) / max(high - low, 1e-3)).clamp(0, 1)
    return w / f * ramp + w * (1 - ramp), 0.1 * math.log(f) + 1.0


def _plain_rope(case, x, pos, w):
    x, rot = x.float(), case["rot"]
    if w is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w
    freq, m = _frequencies(case)
    a = pos.double()[:, None, None] * freq
    cos, sin = (torch.cos(a) * m).float(), (torch.sin(a) * m).float()
    a, b = (x[..., :rot // 2], x[..., rot // 2:rot]) if case["half"] else (x[..., 0:rot:2], x[..., 1:rot:2])
    a, b = a * cos - b * sin, b * cos + a * sin
    y = torch.cat([a, b], -1) if case["half"] else torch.stack([a, b], -1).flatten(-2)
    return torch.cat([y, x[..., rot:]], -1).to(torch.bfloat16)


def _slots(s, pos, start, rows):
    """Block of the pool and place in it of each row, and whether the row's block keeps older tokens."""
    r = torch.arange(rows, device="cuda")
    seq = torch.searchsorted(start[1:].long(), r, right=True)
    p = pos.long()[seq] + r - start.long()[seq]
    block = s["table"].long()[seq, p // PAGE] * 4 + p % PAGE // BLOCK
    first = pos.long()[seq]
    return block, p % BLOCK, (p // BLOCK == first // BLOCK) & (first % BLOCK > 0)


def _pow2(amax):
    """The smallest power of two that holds amax in 7 bits and a sign."""
    m, e = torch.frexp(amax)
    e = torch.where(amax > 0, e - 7 + (m > 127 / 128), torch.full_like(e, -126)).clamp(-126, 120)
    return torch.ldexp(torch.ones_like(amax), e)


def _plain_write(s, k, v, pos, start, rows):
    codes, scales, kv = s["codes"], s["scales"], k.shape[1]
    block, slot, kept = _slots(s, pos, start, rows)
    x = torch.stack([k, v]).float()
    amax = torch.zeros_like(scales).scatter_reduce_(
        1, block[None, :, None].expand(2, rows, kv), x.abs().amax(-1), "amax")[:, block]
    new = _pow2(amax)
    new = torch.where(kept[None, :, None], torch.maximum(new, scales[:, block]), new)
    # the older tokens of a block whose scale grows: once for each such block, by its first new row
    one = kept & (slot == pos.long()[torch.searchsorted(start[1:].long(), torch.arange(rows, device="cuda"), right=True)] % BLOCK)
    b = block[one]
    codes[:, b] = torch.round(codes[:, b].float() * (scales[:, b] / new[:, one])[:, :, None, :, None]).to(torch.int8)
    codes[:, block, slot] = torch.round(x / new[..., None]).clamp(-127, 127).to(torch.int8)
    scales[:, block] = new


def _plain_read(s, pos, start, rows):
    block, slot, _ = _slots(s, pos, start, rows)
    return list((s["codes"][:, block, slot].float() * s["scales"][:, block][..., None]).to(torch.bfloat16).unbind(0))


def _plain_attn(s):
    n, kv, dim = s["n"], s["case"]["kv"], s["case"]["dim"]
    block = (s["table"].long()[:, :, None] * 4 + torch.arange(4, device="cuda")).flatten(1)         # [n, blocks]
    q = s["q"].float().unflatten(1, (kv, -1))
    k = s["codes"][0][block].float() * s["scales"][0][block][:, :, None, :, None]                   # [n, b, 16, kv, dim]
    a = torch.einsum("nhgd,nbthd->nhgbt", q, k).flatten(3) * s["scale"]
    del k
    there = torch.arange(a.shape[3], device="cuda") < s["len"].long()[:, None, None, None]
    a = a.masked_fill(~there, -math.inf)
    p = torch.exp(a - a.amax(-1, keepdim=True).clamp(min=-1e38)) * there
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-30)
    v = s["codes"][1][block].float() * s["scales"][1][block][:, :, None, :, None]
    o = torch.einsum("nhgbt,nbthd->nhgd", p.unflatten(3, (-1, BLOCK)), v).flatten(1, 2)
    if s["gate"] is not None:
        o = o / (1 + torch.exp(-s["gate"].float()))
    return [o.to(torch.bfloat16)]


# ------------------------------------------------------- work and 64 bits

def work(case):
    if case["op"] == "rope":
        values = case["rows"] * (case["nq"] + case["nk"]) * case["dim"]
        return {"bytes": 4 * values + 4 * case["rows"], "flops": 6 * values}
    values = int(_lengths(case).sum()) * case["kv"] * case["dim"] * 2   # K and V
    if case["op"] == "write":                                       # rows in, codes out; codes in, values out
        back = values + int((_starts(case) % BLOCK).sum()) * case["kv"] * case["dim"] * 2
        return {"bytes": 3 * values + 3 * back, "flops": 4 * values}
    heads = case["n"] * case["kv"] * case["group"] * case["dim"]
    return {"bytes": int(values + values / case["dim"] / BLOCK * 4 + heads * (6 if case["gate"] else 4)),
            "flops": 2 * values * case["group"]}


def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "rope":
        return [_exact_rope(case, s["q"], s["pos"], s.get("qw")), _exact_rope(case, s["k"], s["pos"], s.get("kw"))]
    if case["op"] == "write":
        return [_exact_write(s, s["old_k"], s["k"]), _exact_write(s, s["old_v"], s["v"])]
    return [_exact_attn(case, s)]


def _exact_rope(case, x, pos, w):
    """The rotation as a product of complex numbers."""
    y, rot, f = x.double(), case["rot"], case["factor"]
    if w is not None:
        y = y / (y.pow(2).sum(-1, keepdim=True) / case["dim"] + EPS).sqrt() * w.double()
    base = case["base"] * (f ** (rot / (rot - 2)) if case["scaling"] == "ntk" else 1.0)
    w = np.array([base ** -(2 * i / rot) for i in range(rot // 2)])
    size = 1.0
    if case["scaling"] == "linear":
        w = w / f
    if case["scaling"] == "yarn":
        edge = [rot / 2 * (math.log(case["orig"]) - math.log(2 * math.pi * b)) / math.log(base) for b in (32.0, 1.0)]
        lo, hi = max(0, math.floor(edge[0])), min(rot - 1, math.ceil(edge[1]))
        share = np.clip((np.arange(rot // 2) - lo) / max(hi - lo, 1e-3), 0, 1)
        w, size = w * (1 - share + share / f), 1 + math.log(f) / 10
    turn = torch.polar(torch.full((1,), size, dtype=torch.float64, device="cuda"),
                       pos.double()[:, None] * torch.from_numpy(w).cuda())[:, None]
    head = y[..., :rot].unflatten(-1, (2, -1)).transpose(-1, -2) if case["half"] else y[..., :rot].unflatten(-1, (-1, 2))
    z = torch.view_as_real(torch.view_as_complex(head.contiguous()) * turn)
    y[..., :rot] = (z.transpose(-1, -2) if case["half"] else z).flatten(-2)
    return y


def _exact_scale(x, dims=(0, 2)):
    """2^ceil(log2(largest magnitude / 127)) over a block's tokens and dims.  Neighbouring bf16 values are a factor of
    1 + 2^-7 apart at the least, so the 1e-9 only keeps log2's own error at whole numbers out of it."""
    return torch.exp2(torch.ceil(torch.log2(x.abs().amax(dims, keepdim=True).clamp(min=127 * 2.0 ** -126) / 127) - 1e-9))


def _exact_write(s, old, new):
    old, new, outs = old.double(), new.double(), []
    os_, ns, pos = s["old_start"].tolist(), s["start"].tolist(), s["pos"].tolist()
    for i in range(s["n"]):
        a, x = old[os_[i]:os_[i + 1]], new[ns[i]:ns[i + 1]]
        lead = min(len(x), (-pos[i]) % BLOCK)
        if len(a):      # quantised when it was written, and again if the block's scale grows
            sc = _exact_scale(a)
            a = torch.round(a / sc) * sc
            big = torch.maximum(sc, _exact_scale(x[:lead])) if lead else sc
            outs += [torch.round(a / big) * big, torch.round(x[:lead] / big) * big]
            x = x[lead:]
        full = x[:len(x) // BLOCK * BLOCK].unflatten(0, (-1, BLOCK))
        if len(full):
            sc = _exact_scale(full, (1, 3))
            outs.append((torch.round(full / sc) * sc).flatten(0, 1))
        tail = x[len(x) // BLOCK * BLOCK:]
        if len(tail):
            sc = _exact_scale(tail)
            outs.append(torch.round(tail / sc) * sc)
    return torch.cat(outs)


def _exact_attn(case, s):
    n, kv, dim, heads = s["n"], case["kv"], case["dim"], s["heads"]
    out = torch.zeros(n, heads, dim, dtype=torch.float64, device="cuda")
    start = s["start"].tolist()
    for i in range(n):
        lo, hi = start[i], start[i + 1]
        if hi == lo:
            continue
        deq = []
        for x in (s["k"], s["v"]):
            x = x[lo:hi].double()
            x = torch.cat([x, x.new_zeros((-len(x)) % BLOCK, kv, dim)]).unflatten(0, (-1, BLOCK))
            sc = _exact_scale(x, (1, 3))
            deq.append((torch.round(x / sc) * sc).flatten(0, 1)[:hi - lo].transpose(0, 1))
        q = s["q"][i].double().unflatten(0, (kv, -1))
        p = torch.softmax(q @ deq[0].transpose(1, 2) * s["scale"], -1)
        out[i] = (p @ deq[1]).flatten(0, 1)
    return out * torch.sigmoid(s["gate"].double()) if s["gate"] is not None else out
