"""The operators of a 4-bit K/V cache, as timed cases.

A serving engine that keeps its paged K/V cache in MXFP4 (OCP MX: E2M1 codes, one
power-of-two scale per 32 values of a row) calls per layer and step

  append   RMS norm of every query and key head (optional), NeoX rotation, and the
           new K/V rows written into their pages, quantised or as BF16
  decode   paged batch decode attention over the MXFP4 pages
  read     rows of the cache read back as BF16, contiguous per request: the prefix
           of a chunked prompt, for a ragged prefill

The append cases on MXFP4 pages read the rows that they wrote back, so that their
outputs are the values the cache holds.  `own` selects the library's commands;
without it every operator is computed from elementary torch operations.
"""
import math
import os
import random
import sys

import numpy as np
import torch

own = False

D = 128
BLOCK = 32  # values of a row that share a scale
MAX_COMMANDS = 1 << 40
THETA = 1000000.0
EPS = 1e-6
LN2 = math.log(2.0)


def listed():
    return [
        # Decode: one chat's next token, some hundred tokens of context (latency).
        _case("decode_b1_200", "decode", 1, 200, 200, 32, 8),
        # A chat server at moderate load: 16 requests of some hundred tokens.
        _case("decode_b16_1k", "decode", 16, 256, 1536, 32, 8),
        # The headline decode: 64 ragged requests, context U[512, 8192], GQA4.
        _case("decode_b64_ragged", "decode", 64, 512, 8192, 32, 8, page=64, layout="HND"),
        # Long documents: 8 requests of 32768 tokens, GQA8.
        _case("decode_b8_32k", "decode", 8, 32768, 32768, 64, 8, page=32),
        # Seven query heads per kv-head, lengths from one token on, 16-row pages.
        _case("decode_b5_odd", "decode", 5, 1, 5003, 28, 4, layout="HND"),
        # Append: one new token of each of 64 requests, normed (a decode step).
        _case("append_step_b64", "append", 64, 16, 512, 32, 8, rows_lo=1, rows_hi=1, norm=True),
        # Chunks of 32 prompts, about 1000 tokens in one command, without norms.
        _case("append_chunks_b32", "append", 32, 64, 512, 32, 8, rows_lo=1, rows_hi=64, page=32),
        # The most tokens that one command takes: a long prompt's chunk, normed.
        _case("append_8192", "append", 2, 4096, 4096, 64, 8, rows_lo=4096, rows_hi=4096, norm=True,
              layout="HND", page=64),
        # Norms and rotation into BF16 pages: one new token of four chats.
        _case("norm_rope_b4", "append", 4, 3, 41, 16, 4, rows_lo=1, rows_hi=1, norm=True, dtype="bf16"),
        # The same of about 1000 tokens of 32 prompts.
        _case("norm_rope_b32", "append", 32, 64, 512, 32, 8, rows_lo=1, rows_hi=64, norm=True,
              dtype="bf16"),
        # Read back: a short prefix of odd length.
        _case("read_b1_777", "read", 1, 777, 777, 16, 4),
        # The prefixes of 4 long prompts that go on in chunks.
        _case("read_b4_16k", "read", 4, 2048, 16384, 32, 8, layout="HND", page=64),
    ]


def _case(name, op, batch, lo, hi, hq, hkv, page=16, layout="NHD", dtype="mxfp4", rows_lo=0,
          rows_hi=0, norm=False, mix=7):
    case = dict(op=op, batch=batch, lo=lo, hi=hi, hq=hq, hkv=hkv, page=page, layout=layout,
                dtype=dtype, rows_lo=rows_lo, rows_hi=rows_hi, norm=norm, mix=mix)
    return case if name is None else dict(name=name, **case)


# Query and kv heads of the repository's configurations and fixtures, and one odd group.
HEADS = [(32, 8), (32, 8), (64, 8), (16, 4), (32, 32), (8, 1), (28, 4)]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case: sizes log-uniform over what the listed cases span, within the
    largest one's K/V tokens."""
    op = rng.choice(["decode", "decode", "append", "append", "read"])
    hq, hkv = rng.choice(HEADS)
    form = dict(page=rng.choice([16, 16, 32, 64]), layout=rng.choice(["NHD", "HND"]),
                mix=rng.randrange(1 << 20))
    most = (1 << 21) // hkv if op == "decode" else (1 << 18) // hkv  # K/V tokens of the call
    if op == "append":
        b = _log(rng, 1, 128)
        rows = max(1, min(2048, 4096 // b, _log(rng, 1, 2048)))
        lo = rows + _log(rng, 1, 64)
        return _case(None, op, b, lo, lo + _log(rng, 16, 512), hq, hkv, rows_lo=max(1, rows // 8),
                     rows_hi=rows, norm=rng.random() < 0.6,
                     dtype=rng.choice(["mxfp4", "mxfp4", "bf16"]), **form)
    b = _log(rng, 1, 128)
    hi = max(16, min(_log(rng, 16, 32768), most // b))
    lo = max(1, int(hi * rng.choice([0.06, 0.5, 1.0])))
    return _case(None, op, b, lo, hi, hq, hkv, **form)


# ---- lengths and tables ---------------------------------------------------------
def _lengths(case):
    """(K/V length, new rows) of every request: the case's own, whatever the inputs'
    seed.  The longest and the shortest of the range are among them."""
    r = random.Random(case["mix"])
    b, lo, hi = case["batch"], case["lo"], case["hi"]
    lens = [r.randint(lo, hi) for _ in range(b)]
    lens[0] = hi
    lens[-1] = lo if b > 1 else hi
    rows = [min(n, r.randint(case["rows_lo"], case["rows_hi"])) for n in lens]
    if case["op"] == "read":
        rows = list(lens)  # whole contexts
    return lens, rows


def _table(case, lens, rng):
    """Every request's pages scattered over a pool an eighth larger than they need."""
    P = case["page"]
    pages = [-(-n // P) for n in lens]
    indptr = np.concatenate([[0], np.cumsum(pages)]).astype(np.int32)
    total = int(indptr[-1])
    pool = total + max(4, total // 8)
    indices = rng.permutation(pool)[:total].astype(np.int32)
    last = np.array([n - (p - 1) * P for n, p in zip(lens, pages)], np.int32)
    return pool, indptr, indices, last


def _starts(counts):
    return np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)


def _random_cache(pool, P, hkv, layout, g):
    """Codes and scales of a cache whose rows were normal with a spread of their own
    (0.5 to 2 per page and head), quantised in 32 bits (exact: scales are powers of two)."""
    codes = torch.empty((pool, P, hkv, D // 2) if layout == "NHD" else (pool, hkv, P, D // 2),
                        dtype=torch.uint8, device="cuda")
    scales = torch.empty((pool, hkv, P, D // BLOCK), dtype=torch.uint8, device="cuda")
    edges = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device="cuda")
    step = max(1, (1 << 26) // (P * hkv * D))
    for a in range(0, pool, step):
        z = min(pool, a + step)
        x = torch.randn((z - a, hkv, P, D // BLOCK, BLOCK), generator=g, device="cuda")
        x *= torch.exp2(torch.rand((z - a, hkv, 1, 1, 1), generator=g, device="cuda") * 2 - 1)
        e = torch.frexp(x.abs().amax(-1, keepdim=True))[1] - 3
        c = torch.bucketize(torch.ldexp(x.abs(), -e), edges) + 8 * (x < 0)
        c = c.to(torch.uint8).flatten(-2)
        c = c[..., 0::2] | (c[..., 1::2] << 4)
        codes[a:z] = c if layout == "HND" else c.transpose(1, 2)
        scales[a:z] = (e[..., 0] + 127).to(torch.uint8)
    return codes, scales


def _inputs(case, seed):
    """The inputs of one call on the GPU, from the seed alone."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    rng = np.random.default_rng(seed)

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda", dtype=torch.bfloat16)

    def ints(a):
        return torch.from_numpy(np.ascontiguousarray(np.asarray(a, np.int32))).cuda()

    hq, hkv, P, op = case["hq"], case["hkv"], case["page"], case["op"]
    lens, rows = _lengths(case)
    pool, indptr, indices, last = _table(case, lens, rng)
    x = {"pool": pool, "longest": max(lens), "n": sum(rows),
         "indptr": ints(indptr), "indices": ints(indices), "last": ints(last)}
    if case["dtype"] == "mxfp4":
        x["kp"], x["ks"] = _random_cache(pool, P, hkv, case["layout"], g)
        x["vp"], x["vs"] = _random_cache(pool, P, hkv, case["layout"], g)
    else:
        shape = (pool, P, hkv, D) if case["layout"] == "NHD" else (pool, hkv, P, D)
        x["kp"], x["vp"] = normal(*shape), normal(*shape)
    if op == "decode":
        x["q"] = normal(case["batch"], hq, D)
        return x
    n = sum(rows)
    # the rows to read back: each request's last ones (whole contexts for "read")
    x["kv_indptr"] = ints(_starts(rows))
    x["kv_start"] = ints([a - r for a, r in zip(lens, rows)])
    if op == "append":
        # each request's new tokens at the end of its pages, in a scheduler's mixed order
        req = np.repeat(np.arange(len(lens)), rows)
        pos = np.concatenate([np.arange(a - r, a) for a, r in zip(lens, rows)])
        order = rng.permutation(n)
        x["req"], x["pos"] = ints(req[order]), ints(pos[order])
        x["q"], x["nk"], x["nv"] = normal(n, hq, D), normal(n, hkv, D), normal(n, hkv, D)
        # a projection's outputs: heads and channels of unlike size
        x["nk"] *= torch.exp2(torch.randn(hkv, D, generator=g, device="cuda")).to(torch.bfloat16)
        if case["norm"]:
            x["qw"], x["kw"] = (1 + 0.25 * normal(D) for _ in range(2))
    return x


# ---- a user's program -------------------------------------------------------------
class _Program:
    """What a caller keeps: outputs, plans, queue, bindings and the open scope that
    its commands go into."""

    def __init__(self, case, x):
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                                        "loom-kernels_amd"))
        import loom_infer_hip as L

        op, hq, hkv, b = case["op"], case["hq"], case["hkv"], case["batch"]
        form = dict(kv_layout=case["layout"], kv_dtype=case["dtype"], kv_page_size=case["page"])
        mx = case["dtype"] == "mxfp4"
        self.queue = L.CommandQueue(torch.cuda.current_stream(), MAX_COMMANDS)
        self.commands, self.out = [], {}
        bd = self.queue.bindings(24)
        table = [bd.bind_read(x[k]) for k in ("indptr", "indices", "last")]
        if op == "decode":
            o = torch.zeros(b, hq, D, device="cuda", dtype=torch.bfloat16)
            lse = torch.zeros(b, hq, device="cuda")
            plan = L.DecodeProvider.load(0).plan_bf16_paged_batch(
                L.Bf16PagedBatchDecodeSpec(b, x["pool"], hq, hkv, **form))
            self.queue.reserve_workspace(plan.workspace_bytes)
            q, kp, vp, ks, vs = (bd.bind_read(x[k]) for k in ("q", "kp", "vp", "ks", "vs"))
            ho, hl = bd.bind_read_write(o), bd.bind_read_write(lse)
            self.commands.append((plan, L.Mxfp4PagedBatchDecodeArgs(
                q, kp, vp, ks, vs, *table, ho.write(), hl.write())))
            self.out = {"out": o, "lse": lse}
        else:
            pages = [bd.bind_read_write(x[k]) for k in (("kp", "vp", "ks", "vs") if mx else ("kp", "vp"))]
        if op == "append":
            n = x["q"].shape[0]
            qo = torch.zeros(n, hq, D, device="cuda", dtype=torch.bfloat16)
            spec = L.NormRopePagedKvAppendSpec(n, b, x["pool"], hq, hkv, rope_theta=THETA,
                                               norm_eps=EPS if case["norm"] else None, **form)
            q, nk, nv, req, pos = (bd.bind_read(x[k]) for k in ("q", "nk", "nv", "req", "pos"))
            more = {}
            if mx:
                more = dict(key_scales=pages[2].write(), value_scales=pages[3].write())
            if case["norm"]:
                more |= dict(query_norm=bd.bind_read(x["qw"]), key_norm=bd.bind_read(x["kw"]))
            self.commands.append((L.RopeProvider.load(0).plan_norm_paged_append(spec),
                                  L.NormRopePagedKvAppendArgs(
                q, nk, nv, *table, bd.bind_read_write(qo).write(), pages[0].write(),
                pages[1].write(), batch_indices=req, positions=pos, **more)))
            self.out = {"q": qo} if mx else {"q": qo, "k_pages": x["kp"], "v_pages": x["vp"]}
        if op == "read" or (op == "append" and mx):
            k, v = (torch.zeros(x["n"], hkv, D, device="cuda", dtype=torch.bfloat16) for _ in range(2))
            plan = L.PrefillProvider.load(0).plan_paged_kv_read(
                L.PagedKvReadSpec(b, x["n"], x["pool"], hkv, **form))
            rk, rv = bd.bind_read_write(k), bd.bind_read_write(v)
            self.commands.append((plan, L.PagedKvReadArgs(
                *(p.read() for p in pages), *table, bd.bind_read(x["kv_indptr"]), rk.write(),
                rv.write(), kv_start=bd.bind_read(x["kv_start"]))))
            self.out |= {"k": k, "v": v}
        self.scope = self.queue.begin(bd)

    def __call__(self):
        for plan, args in self.commands:
            plan.enqueue_into(self.scope, args)
        return self.out


def prepare(case, seed):
    x = _inputs(case, seed)
    return {"case": case, "x": x, "program": _Program(case, x) if own else None}


def run(state):
    if own:
        return state["program"]()
    case, x = state["case"], state["x"]
    if case["op"] == "decode":
        return _decode(case, x)
    if case["op"] == "read":
        return _read(case, x)
    return _append(case, x)


# ---- the plain forms ----------------------------------------------------------------
_VALUES = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def _values(codes, scales):
    """The FP32 values of MXFP4 rows: codes [..., 64] (even value in the low nibble)
    and scales [..., 4]."""
    t = torch.tensor(_VALUES + [-v for v in _VALUES], device=codes.device)
    pair = torch.stack([t.repeat(16), t.repeat_interleave(16)], -1)  # byte -> its two values
    v = pair[codes.long()].reshape(*codes.shape[:-1], D // BLOCK, BLOCK)
    return (v * torch.exp2(scales.float() - 127)[..., None]).flatten(-2)


def _page_rows(case, pages, which):
    """The chosen pages as [..., P, Hkv, row]."""
    rows = pages[which]
    return rows.transpose(-3, -2) if case["layout"] == "HND" else rows


def _decode(case, x):
    b, hq, hkv, P = case["batch"], case["hq"], case["hkv"], case["page"]
    most = -(-x["longest"] // P)
    at = x["indptr"][:-1, None] + torch.arange(most, device="cuda")
    which = x["indices"][at.clamp(max=x["indices"].shape[0] - 1).long()].long()
    n = (x["indptr"].diff() - 1) * P + x["last"]

    def rows(codes, scales):  # [B, Hkv, most * P, 128]
        v = _values(_page_rows(case, codes, which), scales[which].transpose(-3, -2))
        return v.reshape(b, most * P, hkv, D).transpose(1, 2).contiguous()

    q = x["q"].float().view(b, hkv, hq // hkv, D)
    s = torch.matmul(q, rows(x["kp"], x["ks"]).transpose(2, 3).contiguous()) * D ** -0.5
    s = s.masked_fill(torch.arange(most * P, device="cuda") >= n[:, None, None, None], -math.inf)
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - m)
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, rows(x["vp"], x["vs"])) / total
    return {"out": out.reshape(b, hq, D).to(torch.bfloat16),
            "lse": ((m + total.log()) / LN2).reshape(b, hq)}


def _slots(case, x, req, pos):
    """(page, row) of each token."""
    return x["indices"][(x["indptr"][req.long()] + pos // case["page"]).long()].long(), \
        (pos % case["page"]).long()


def _read(case, x):
    t = torch.arange(x["n"], device="cuda", dtype=torch.int32)
    req = torch.searchsorted(x["kv_indptr"], t, right=True) - 1
    page, row = _slots(case, x, req, x["kv_start"][req] + t - x["kv_indptr"][req])
    got = {}
    for name, codes, scales in (("k", x["kp"], x["ks"]), ("v", x["vp"], x["vs"])):
        c = codes[page, :, row] if case["layout"] == "HND" else codes[page, row]
        got[name] = _values(c, scales[page, :, row]).to(torch.bfloat16)
    return got


def _normed_rotated(x, w, pos, dtype):
    """RMS norm of every head by weights w (none: not normed) and NeoX rotation of
    x [T, H, 128], computed in `dtype`; angles in 64 bits."""
    y = x.to(dtype)
    if w is not None:
        y = y * (y.square().mean(-1, keepdim=True) + EPS).rsqrt() * w.to(dtype)
    inv = THETA ** (-torch.arange(0, D, 2, device=x.device, dtype=torch.float64) / D)
    a = pos.double()[:, None, None] * inv
    c, s = a.cos().to(dtype), a.sin().to(dtype)
    y1, y2 = y[..., : D // 2], y[..., D // 2:]
    return torch.cat([y1 * c - y2 * s, y2 * c + y1 * s], -1)


def _quantised(v):
    """MXFP4 codes [..., 64] and scales [..., 4] of rows v [..., 128] in 64 bits: of each
    block of 32 the scale 2^(floor(log2 max) - 2), values rounded to nearest even."""
    v = v.unflatten(-1, (D // BLOCK, BLOCK))
    e = (torch.frexp(v.abs().amax(-1, keepdim=True))[1].long() - 3).clamp(-126, 125)
    u = v.abs() * ((1023 - e) << 52).view(torch.float64)
    c = ((u > 0.25).to(torch.uint8) + (u >= 0.75) + (u > 1.25) + (u >= 1.75) + (u > 2.5)
         + (u >= 3.5) + (u > 5.0) + 8 * torch.signbit(v)).to(torch.uint8).flatten(-2)
    return c[..., 0::2] | (c[..., 1::2] << 4), (e[..., 0] + 127).to(torch.uint8)


def _append(case, x):
    pos, mx = x["pos"], case["dtype"] == "mxfp4"
    q = _normed_rotated(x["q"], x.get("qw"), pos, torch.float32).to(torch.bfloat16)
    # which of two codes a key gets hangs on values next to a border: 64 bits
    k = _normed_rotated(x["nk"], x.get("kw"), pos, torch.float64 if mx else torch.float32)
    page, row = _slots(case, x, x["req"], pos)

    def put(pages, rows):
        if case["layout"] == "HND":
            pages[page, :, row] = rows
        else:
            pages[page, row] = rows

    if not mx:
        put(x["kp"], k.to(torch.bfloat16))
        put(x["vp"], x["nv"])
        return {"q": q, "k_pages": x["kp"], "v_pages": x["vp"]}
    for codes, scales, rows in (("kp", "ks", k), ("vp", "vs", x["nv"].double())):
        c, e = _quantised(rows)
        put(x[codes], c)
        x[scales][page, :, row] = e
    return {"q": q, **_read(case, x)}


# ---- what a pass cannot do without ----------------------------------------------
def work(case):
    hq, hkv, P = case["hq"], case["hkv"], case["page"]
    lens, rows = _lengths(case)
    n, tokens = sum(rows), sum(lens)
    row = D // 2 + D // BLOCK if case["dtype"] == "mxfp4" else 2 * D  # one head's K or V row in a page
    table = 4 * (2 * len(lens) + 1)
    if case["op"] == "decode":
        return {"bytes": 2 * tokens * hkv * row + len(lens) * hq * (4 * D + 4) + table
                + 4 * sum(-(-t // P) for t in lens), "flops": 4 * D * hq * tokens}
    # rows read back: their page rows, BF16 rows out, the page indices of the rows
    back = 2 * n * hkv * (row + 2 * D) + table + 8 * len(lens) + 4 * -(-n // P)
    if case["op"] == "read":
        return {"bytes": back, "flops": 2 * n * hkv * D}
    new = n * (hq * 4 * D + 2 * hkv * (2 * D + row)) + 8 * n + table
    flops = (3 + 4 * case["norm"]) * n * (hq + hkv) * D
    return {"bytes": new + (back if case["dtype"] == "mxfp4" else 0), "flops": flops}


# ---- the same in 64 bits ----------------------------------------------------------
def _value64(codes, scales):
    """MXFP4 rows from the bits of their codes: sign, two exponent bits, one mantissa bit."""
    n = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).to(torch.int64)
    ex, mant = (n >> 1) & 3, (n & 1).double()
    v = torch.where(ex > 0, (1 + mant / 2) * torch.exp2((ex - 1).double()), mant / 2)
    v = torch.where(n > 7, -v, v)
    return v * torch.exp2(scales.double() - 127).repeat_interleave(BLOCK, -1)


def _request(case, x, codes, scales, r, n):
    """Request r's first n rows [n, Hkv, 128] out of its pages."""
    ip = x["indptr"].tolist()
    pages = x["indices"][ip[r]:ip[r + 1]].long()
    c = codes[pages] if case["layout"] == "HND" else codes[pages].transpose(1, 2)
    return _value64(c, scales[pages]).transpose(1, 2).reshape(-1, case["hkv"], D)[:n]


def _rotate64(y, pos):
    a = pos.double()[:, None] * torch.exp(
        torch.arange(D // 2, device=y.device, dtype=torch.float64) * (-2 * math.log(THETA) / D))
    z = torch.polar(torch.ones_like(a), a)[:, None] * torch.complex(y[..., : D // 2], y[..., D // 2:])
    return torch.cat([z.real, z.imag], -1)


def _nearest64(v):
    """The MXFP4 values nearest to rows v (ties to the even code), block by block."""
    b = v.reshape(-1, BLOCK)
    grid = torch.tensor(_VALUES, device=v.device, dtype=torch.float64)
    big = b.abs().amax(1, keepdim=True)
    e = torch.floor(torch.log2(torch.where(big > 0, big, torch.ones_like(big))))
    # log2 of a value just under a power of two may round up to it
    e = torch.where(torch.exp2(e) > big, e - 1, e) - 2
    e = torch.where(big > 0, e.clamp(-126, 125), torch.full_like(e, -126))
    u = b.abs() * torch.exp2(-e)
    lo = (torch.searchsorted(grid, u.contiguous(), right=True) - 1).clamp(0, 7)
    hi = (lo + 1).clamp(max=7)
    down, up = u - grid[lo], grid[hi] - u
    code = torch.where((down < up) | ((down == up) & (lo % 2 == 0)), lo, hi)
    return (grid[code] * torch.exp2(e) * torch.where(b < 0, -1.0, 1.0).double()).reshape(v.shape)


def exact(case, seed):
    x = _inputs(case, seed)
    lens, rows = _lengths(case)
    hq, hkv = case["hq"], case["hkv"]
    if case["op"] == "decode":
        out = torch.empty(len(lens), hq, D, device="cuda", dtype=torch.float64)
        lse = out.new_empty(len(lens), hq)
        for r, n in enumerate(lens):
            k, v = (_request(case, x, x[c], x[s], r, n) for c, s in (("kp", "ks"), ("vp", "vs")))
            for h in range(hkv):
                heads = slice(h * (hq // hkv), (h + 1) * (hq // hkv))
                s = k[:, h].contiguous() @ x["q"][r, heads].double().t().contiguous() / math.sqrt(D)
                lse[r, heads] = torch.logsumexp(s, 0) / LN2
                out[r, heads] = torch.softmax(s, 0).t().contiguous() @ v[:, h].contiguous()
        return {"out": out, "lse": lse}
    if case["op"] == "read":
        k, v = (torch.cat([_request(case, x, x[c], x[s], r, n) for r, n in enumerate(lens)])
                for c, s in (("kp", "ks"), ("vp", "vs")))
        return {"k": k, "v": v}
    pos = x["pos"]

    def head(t, w):
        y = t.double()
        if w is not None:
            y = y * w.double() / torch.sqrt((y * y).sum(-1, keepdim=True) / D + EPS)
        return _rotate64(y, pos)

    q, k, v = head(x["q"], x.get("qw")), head(x["nk"], x.get("kw")), x["nv"].double()
    if case["dtype"] == "mxfp4":
        # rows in the order of the requests, as they are read back
        order = torch.argsort(x["req"].long() * (1 << 32) + pos.long())
        return {"q": q, "k": _nearest64(k)[order], "v": _nearest64(v)[order]}
    kp, vp = x["kp"].double(), x["vp"].double()
    ip, ix = x["indptr"].tolist(), x["indices"].tolist()
    slot = [(ix[ip[r] + t // case["page"]], t % case["page"])
            for r, t in zip(x["req"].tolist(), pos.tolist())]
    page, row = (torch.tensor(a, device="cuda") for a in zip(*slot))
    for pages, new in ((kp, k), (vp, v)):
        if case["layout"] == "HND":
            pages[page, :, row] = new
        else:
            pages[page, row] = new
    return {"q": q, "k_pages": kp, "v_pages": vp}
