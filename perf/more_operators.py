"""Attention with a sliding window and sinks over a paged K/V cache, as timed cases.

A serving engine calls these for every layer whose rows see the request's first `sinks`
tokens and the last `window` ones (window 0: the whole prefix):

  decode   one new token of every request
  chunk    ragged rows of new tokens behind each request's cached prefix

over BF16, FP8 E4M3 or MXFP4 pages.  An engine may give the pages that no row sees any
more to other requests; their entries of the page table are -1 then (`freed`).  `own`
selects the library's commands; without it every operator is computed from elementary
torch operations.
"""
import math
import os
import random
import sys

import numpy as np
import torch

own = False

D = 128
BLOCK = 32  # values of an MXFP4 row that share a scale
LN2 = math.log(2.0)
MAX_COMMANDS = 1 << 40
K_SCALE, V_SCALE = 0.0171, 0.0157  # FP8 pages: N(0, 1) values reach 4.5 sigma below 448


def listed():
    return [
        # One chat's next token with a short window: launch and latency.
        _case("decode_b1_w128", "decode", 1, 300, 300, 32, 8, 128, 4),
        # A chat server at moderate load, windows of 1024.
        _case("decode_b16_w1k", "decode", 16, 256, 8192, 32, 8, 1024, 4),
        # 64 ragged requests, windows of 4096; pages behind the windows given back.
        _case("decode_b64_w4k", "decode", 64, 512, 32768, 32, 8, 4096, 4, page=64, layout="HND",
              freed=True),
        # Long documents on FP8 pages, GQA8.
        _case("decode_b8_w8k_fp8", "decode", 8, 32768, 32768, 64, 8, 8192, 16, dtype="fp8_e4m3",
              page=32),
        # A 4-bit cache, seven query heads per kv-head, odd lengths from one token on.
        _case("decode_b24_w2k_mx4", "decode", 24, 1, 9001, 28, 4, 2047, 5, dtype="mxfp4"),
        # Draft verification: 4-8 new rows of each of 16 requests.
        _case("chunk_verify_b16_w1k", "chunk", 16, 1024, 8192, 32, 8, 1024, 4, rows_lo=4, rows_hi=8),
        # A whole 8192-token prompt with a window of 1024.
        _case("chunk_8192_w1k", "chunk", 1, 8192, 8192, 32, 8, 1024, 4, rows_lo=8192, rows_hi=8192),
        # Eight prompts of odd lengths under a short window.
        _case("chunk_b8_w128", "chunk", 8, 200, 2047, 16, 4, 128, 1, rows_lo=2047, rows_hi=2047,
              layout="HND"),
        # Chunks of four long prompts on FP8 pages, windows of 4096.
        _case("chunk_b4_w4k_fp8", "chunk", 4, 2048, 16384, 32, 8, 4096, 4, rows_lo=512, rows_hi=512,
              dtype="fp8_e4m3", freed=True),
        # The same chunks over a 4-bit cache and the whole prefix.
        _case("chunk_b4_mx4", "chunk", 4, 2048, 16384, 32, 8, 0, 0, rows_lo=512, rows_hi=512,
              dtype="mxfp4", layout="HND", page=64),
        # A few new rows of eight conversations over a 4-bit cache and the whole prefix.
        _case("chunk_b8_rows_mx4", "chunk", 8, 300, 5000, 32, 8, 0, 0, rows_lo=1, rows_hi=32,
              dtype="mxfp4"),
        # The largest: a long prompt over a 4-bit cache, window 4096.
        _case("chunk_16k_w4k_mx4", "chunk", 1, 16384, 16384, 32, 8, 4096, 4, rows_lo=16384,
              rows_hi=16384, dtype="mxfp4", page=64),
    ]


def _case(name, op, batch, lo, hi, hq, hkv, window, sinks, page=16, layout="NHD", dtype="bf16",
          rows_lo=1, rows_hi=1, freed=False, mix=7):
    case = dict(op=op, batch=batch, lo=lo, hi=hi, hq=hq, hkv=hkv, window=window, sinks=sinks,
                page=page, layout=layout, dtype=dtype, rows_lo=rows_lo, rows_hi=rows_hi,
                freed=freed, mix=mix)
    return case if name is None else dict(name=name, **case)


# Query and kv heads of the repository's configurations and fixtures, and one odd group.
HEADS = [(32, 8), (32, 8), (64, 8), (16, 4), (32, 32), (8, 1), (28, 4)]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case: sizes log-uniform over what the listed cases span, within the
    largest ones' K/V tokens and products."""
    hq, hkv = rng.choice(HEADS)
    dtype = rng.choice(["bf16", "bf16", "fp8_e4m3", "mxfp4", "mxfp4"])
    form = dict(page=rng.choice([16, 16, 32, 64]), layout=rng.choice(["NHD", "HND"]), dtype=dtype,
                mix=rng.randrange(1 << 20))
    sinks = rng.choice([0, 1, 4, 4, rng.randint(0, 100)])
    if rng.random() < 0.5:
        b = _log(rng, 1, 128)
        window = max(1, min(_log(rng, 16, 8192), (1 << 21) // (b * hkv)))
        hi = max(4, min(_log(rng, 64, 32768), (1 << 22) // (b * hkv)))
        lo = max(1, int(hi * rng.choice([0.01, 0.3, 1.0])))
        return _case(None, "decode", b, lo, hi, hq, hkv, window, sinks, freed=rng.random() < 0.5,
                     **form)
    b = _log(rng, 1, 32)
    rows = max(1, min(_log(rng, 1, 8192), 16384 // b))
    window = _log(rng, 16, 8192)
    if dtype == "mxfp4" and rng.random() < 0.5:
        window = sinks = 0
    hi = max(rows, min(rows + _log(rng, 1, 16384), 65536 // b))
    # products: rows * seen tokens * query heads
    while b * rows * min(hi, window or hi) * hq > 1 << 31 and rows > 1:
        rows = max(1, rows // 2)
    lo = max(1, int(hi * rng.choice([0.06, 0.5, 1.0])))
    return _case(None, "chunk", b, lo, hi, hq, hkv, window, sinks,
                 rows_lo=max(1, int(rows * rng.choice([0.1, 0.5, 1.0]))), rows_hi=rows,
                 freed=window > 0 and rng.random() < 0.3, **form)


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
    return lens, rows


def _first(case, n, rows):
    """First token that the request's first row sees in its window."""
    return max(0, n - rows + 1 - case["window"]) if case["window"] else 0


def _table(case, rng):
    """Every request's pages scattered over a pool an eighth larger than they need."""
    P, S = case["page"], case["sinks"]
    lens, rows = _lengths(case)
    pages = [-(-n // P) for n in lens]
    indptr = np.concatenate([[0], np.cumsum(pages)]).astype(np.int32)
    kept = np.ones(int(indptr[-1]), bool)
    if case["freed"]:
        for r, (n, m) in enumerate(zip(lens, rows)):
            kept[indptr[r] + -(-S // P):indptr[r] + _first(case, n, m) // P] = False
    total = int(kept.sum())
    pool = total + max(4, total // 8)
    indices = np.full(len(kept), -1, np.int32)
    indices[kept] = rng.permutation(pool)[:total]
    last = np.array([n - (p - 1) * P for n, p in zip(lens, pages)], np.int32)
    return pool, indptr, indices, last


def _random_pages(case, pool, lean, g):
    """Codes (or values) of a pool's pages, and the MXFP4 scales: normal rows, a quarter of
    each row's variance shared by all rows of a head (`lean` [Hkv, 128])."""
    P, hkv, dtype = case["page"], case["hkv"], case["dtype"]
    nhd, mx = case["layout"] == "NHD", dtype == "mxfp4"
    width = D // 2 if mx else D
    pages = torch.empty((pool, P, hkv, width) if nhd else (pool, hkv, P, width), device="cuda",
                        dtype=torch.bfloat16 if dtype == "bf16" else torch.uint8)
    scales = torch.empty((pool, hkv, P, D // BLOCK), dtype=torch.uint8, device="cuda") if mx else None
    edges = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device="cuda")
    step = max(1, (1 << 26) // (P * hkv * D))
    for a in range(0, pool, step):
        z = min(pool, a + step)
        x = torch.randn((z - a, hkv, P, D), generator=g, device="cuda") * 0.75 ** 0.5
        x += lean[:, None]
        if mx:
            x = x.unflatten(-1, (D // BLOCK, BLOCK))
            e = torch.frexp(x.abs().amax(-1, keepdim=True))[1] - 3
            c = (torch.bucketize(torch.ldexp(x.abs(), -e), edges) + 8 * (x < 0)).to(torch.uint8)
            c = c.flatten(-2)
            x = c[..., 0::2] | (c[..., 1::2] << 4)
            scales[a:z] = (e[..., 0] + 127).to(torch.uint8)
        elif dtype == "fp8_e4m3":
            x = (x / K_SCALE).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
        pages[a:z] = x.transpose(1, 2) if nhd else x
    return pages, scales


def _inputs(case, seed):
    """The inputs of one call on the GPU, from the seed alone."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    rng = np.random.default_rng(seed)

    def ints(a):
        return torch.from_numpy(np.ascontiguousarray(np.asarray(a, np.int32))).cuda()

    hq, hkv = case["hq"], case["hkv"]
    lens, rows = _lengths(case)
    pool, indptr, indices, last = _table(case, rng)
    x = {"pool": pool, "indptr": ints(indptr), "indices": ints(indices), "last": ints(last),
         "qo": ints(np.concatenate([[0], np.cumsum(rows)]))}
    lean = torch.randn((2, hkv, D), generator=g, device="cuda") * 0.5
    x["kp"], x["ks"] = _random_pages(case, pool, lean[0], g)
    x["vp"], x["vs"] = _random_pages(case, pool, lean[1], g)
    q = torch.randn((sum(rows), hkv, hq // hkv, D), generator=g, device="cuda")
    x["q"] = (q + 0.5 * lean[0][:, None]).reshape(-1, hq, D).to(torch.bfloat16)
    if case["dtype"] == "fp8_e4m3":
        x["scales"] = torch.tensor([K_SCALE, V_SCALE], device="cuda")
    return x


# ---- a user's program -------------------------------------------------------------
class _Program:
    """What a caller keeps: outputs, plan, queue, bindings and the open scope that its
    commands go into."""

    def __init__(self, case, x):
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                                        "loom-kernels_amd"))
        import loom_infer_hip as L

        chunk = case["op"] == "chunk"
        n = x["q"].shape[0]
        self.out = {"out": torch.zeros_like(x["q"]), "lse": torch.zeros(n, case["hq"], device="cuda")}
        spec = L.WindowPagedAttentionSpec(
            n, case["batch"], x["pool"], case["hq"], case["hkv"], window=case["window"],
            sinks=case["sinks"], explicit_rows=chunk, kv_layout=case["layout"],
            kv_dtype=case["dtype"], kv_page_size=case["page"])
        if chunk:
            self.plan = L.PrefillProvider.load(0).plan_window_paged(spec)
        else:
            self.plan = L.DecodeProvider.load(0).plan_window_paged_batch(spec)
        self.queue = L.CommandQueue(torch.cuda.current_stream(), MAX_COMMANDS)
        bd = self.queue.bindings(16)
        read = {k: bd.bind_read(x[k]) for k in ("q", "kp", "vp", "indptr", "indices", "last", "qo")}
        more = {}
        if chunk:
            more["qo_indptr"] = read["qo"]
        if case["dtype"] == "fp8_e4m3":
            more["kv_scales"] = bd.bind_read(x["scales"])
        if case["dtype"] == "mxfp4":
            more |= dict(key_scales=bd.bind_read(x["ks"]), value_scales=bd.bind_read(x["vs"]))
        self.args = L.WindowPagedAttentionArgs(
            read["q"], read["kp"], read["vp"], read["indptr"], read["indices"], read["last"],
            bd.bind_read_write(self.out["out"]).write(), bd.bind_read_write(self.out["lse"]).write(),
            **more)
        self.scope = self.queue.begin(bd)

    def __call__(self):
        self.plan.enqueue_into(self.scope, self.args)
        return self.out


def prepare(case, seed):
    x = _inputs(case, seed)
    return {"case": case, "x": x, "program": _Program(case, x) if own else None}


def run(state):
    if own:
        return state["program"]()
    case, x = state["case"], state["x"]
    return _decode(case, x) if case["op"] == "decode" else _chunk(case, x)


# ---- the plain forms ----------------------------------------------------------------
_VALUES = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def _rows(case, x, which, page, row):
    """The FP32 K ("k") or V rows [..., Hkv, 128] of slots (page, row)."""
    pages = x[which + "p"]
    v = pages[page, :, row] if case["layout"] == "HND" else pages[page, row]
    if case["dtype"] == "bf16":
        return v.float()
    if case["dtype"] == "fp8_e4m3":
        return v.view(torch.float8_e4m3fn).float() * x["scales"][0 if which == "k" else 1]
    t = torch.tensor(_VALUES + [-a for a in _VALUES], device="cuda")
    pair = torch.stack([t.repeat(16), t.repeat_interleave(16)], -1)  # byte -> its two values
    v = pair[v.long()].reshape(*v.shape[:-1], D // BLOCK, BLOCK)
    return (v * torch.exp2(x[which + "s"][page, :, row].float() - 127)[..., None]).flatten(-2)


def _attend(q, k, v, seen):
    """Softmax attention of q [..., rows, 128] over k, v [..., n, 128] where `seen`."""
    s = torch.matmul(q, k.transpose(-1, -2).contiguous()) * D ** -0.5
    s = s.masked_fill(~seen, -math.inf)
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - m)
    total = p.sum(-1, keepdim=True)
    return torch.matmul(p, v) / total, ((m + total.log()) / LN2).squeeze(-1)


def _decode(case, x):
    b, hq, hkv, P, S = case["batch"], case["hq"], case["hkv"], case["page"], case["sinks"]
    n = (x["indptr"].diff() - 1) * P + x["last"]
    width = min(case["window"] or case["hi"], case["hi"])
    begin = (n - width).clamp(min=0)
    near = begin[:, None] + torch.arange(width, device="cuda")
    far = torch.arange(min(S, case["hi"]), device="cuda").expand(b, -1)
    t = torch.cat([far, near], 1)
    seen = torch.cat([far < begin[:, None], near < n[:, None]], 1)
    at = torch.where(seen, t, begin[:, None])  # a token that the row sees
    page = x["indices"][x["indptr"][:-1, None].long() + at // P].long()
    k, v = (_rows(case, x, c, page, at % P).transpose(1, 2).contiguous() for c in "kv")
    out, lse = _attend(x["q"].float().view(b, hkv, hq // hkv, D), k, v, seen[:, None, None])
    return {"out": out.reshape(b, hq, D).to(torch.bfloat16), "lse": lse.reshape(b, hq)}


def _chunk(case, x):
    hq, hkv, P, S, W = case["hq"], case["hkv"], case["page"], case["sinks"], case["window"]
    g = hq // hkv
    lens, rows = _lengths(case)
    ip = np.concatenate([[0], np.cumsum([-(-n // P) for n in lens])])
    out = torch.empty_like(x["q"])
    lse = torch.empty(x["q"].shape[0], hq, device="cuda")
    r0 = 0
    for r, (n, m) in enumerate(zip(lens, rows)):
        for i in range(0, m, 512):  # 512 rows and the keys that they see at a time
            c = min(512, m - i)
            p0 = n - m + i
            begin = max(0, p0 + 1 - W) if W else 0
            t = torch.cat([torch.arange(min(S, begin), device="cuda"),
                           torch.arange(begin, p0 + c, device="cuda")])
            page = x["indices"][int(ip[r]) + t // P].long()
            k, v = (_rows(case, x, a, page, t % P).transpose(0, 1).contiguous() for a in "kv")
            q = x["q"][r0 + i:r0 + i + c].float().view(c, hkv, g, D).permute(1, 2, 0, 3)
            p = p0 + torch.arange(c, device="cuda")[:, None]
            seen = t <= p
            if W:
                seen &= (t > p - W) | (t < S)
            o, l = _attend(q.reshape(hkv, g * c, D), k, v, seen.repeat(g, 1))
            o = o.view(hkv, g, c, D).permute(2, 0, 1, 3).reshape(c, hq, D)
            out[r0 + i:r0 + i + c] = o.to(torch.bfloat16)
            lse[r0 + i:r0 + i + c] = l.view(hkv, g, c).permute(2, 0, 1).reshape(c, hq)
        r0 += m
    return {"out": out, "lse": lse}


# ---- what a pass cannot do without ----------------------------------------------
def work(case):
    hq, hkv, S, W, P = case["hq"], case["hkv"], case["sinks"], case["window"], case["page"]
    row = {"bf16": 4 * D, "fp8_e4m3": 2 * D, "mxfp4": D + 2 * D // BLOCK}[case["dtype"]]  # K and V
    lens, rows = _lengths(case)
    moved = flops = 0
    for n, m in zip(lens, rows):
        first = _first(case, n, m)
        used = n - first + min(S, first)  # tokens that some row sees
        # row at p sees p + 1 tokens, or its window and the sinks before it
        p = np.arange(n - m, n, dtype=np.int64)
        seen = p + 1
        if W:
            seen = np.minimum(p + 1, W) + np.minimum(S, np.maximum(p + 1 - W, 0))
        flops += 4 * D * hq * int(seen.sum())
        moved += used * hkv * row + m * hq * (4 * D + 4) + 4 * -(-used // P)
    return {"bytes": moved + 12 * len(lens), "flops": flops}


# ---- the same in 64 bits ----------------------------------------------------------
def _value64(codes, scales):
    """MXFP4 rows from the bits of their codes: sign, two exponent bits, one mantissa bit."""
    n = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).to(torch.int64)
    ex, mant = (n >> 1) & 3, (n & 1).double()
    v = torch.where(ex > 0, (1 + mant / 2) * torch.exp2((ex - 1).double()), mant / 2)
    v = torch.where(n > 7, -v, v)
    return v * torch.exp2(scales.double() - 127).repeat_interleave(BLOCK, -1)


def _request(case, x, which, r, n):
    """Request r's n rows [Hkv, n, 128] out of its pages; pages given back: zeros."""
    ip = x["indptr"].tolist()
    held = x["indices"][ip[r]:ip[r + 1]].long()
    p = x[which + "p"][held.clamp(min=0)]
    p = p if case["layout"] == "HND" else p.transpose(1, 2)
    if case["dtype"] == "mxfp4":
        v = _value64(p, x[which + "s"][held.clamp(min=0)])
    elif case["dtype"] == "fp8_e4m3":
        v = p.contiguous().view(torch.float8_e4m3fn).float().double()
        v = v * x["scales"].double()[0 if which == "k" else 1]
    else:
        v = p.double()
    v = torch.where((held < 0)[:, None, None, None], torch.zeros_like(v), v)
    return v.transpose(0, 1).reshape(case["hkv"], -1, D)[:, :n]


def exact(case, seed):
    x = _inputs(case, seed)
    lens, rows = _lengths(case)
    hq, hkv, S, W = case["hq"], case["hkv"], case["sinks"], case["window"]
    g = hq // hkv
    out = torch.empty(sum(rows), hq, D, device="cuda", dtype=torch.float64)
    lse = out.new_empty(sum(rows), hq)
    r0 = 0
    for r, (n, m) in enumerate(zip(lens, rows)):
        k, v = (_request(case, x, c, r, n) for c in "kv")
        t = torch.arange(n, device="cuda")
        for i in range(0, m, 512):
            p = torch.arange(n - m + i, n - m + min(i + 512, m), device="cuda")[:, None]
            behind = p - t
            hidden = (behind < 0) | ((behind >= W) & (t >= S) if W else torch.zeros_like(behind, dtype=torch.bool))
            for h in range(hq):
                at = slice(r0 + i, r0 + i + len(p))
                s = x["q"][at, h].double() @ k[h // g].t().contiguous() / math.sqrt(D)
                s = torch.where(hidden, s.new_tensor(-math.inf), s)
                lse[at, h] = torch.logsumexp(s, 1) / LN2
                out[at, h] = torch.softmax(s, 1) @ v[h // g].contiguous()
        r0 += m
    return {"out": out, "lse": lse}
