"""Window attention's inputs, the operator in 64 bits (numpy) and a runner, for the tests.

Tolerances.  Against the definition in 64 bits over the values that the pages hold:
  * a score is a sum of 128 exact products in FP32, off by at most 128 * 2^-24 of the sum S
    of their magnitudes (times softmax scale and log2 e); LSE is off by as much, and a
    weight's ratio to the normalizer by 2 ln 2 of it;
  * row tiles keep 16 bits of a weight in O's product (2^-15), long tiles 8 (2^-8); the
    normalizer sums the weights before that rounding;
  * v_exp_f32 and v_log_f32 are good to about 2^-22 of their results, FP32 sums of n weights
    and products to n * 2^-24 of the sum of their magnitudes;
  * O is rounded once to BF16 (2^-8 of it).
With A = sum |p v| / sum p per dimension: |dO| <= 2^-8 |O| + (weights) A.
"""
import numpy as np

import mxfp4_util as mx

D = 128
LOG2E = 1.4426950408889634
K_SCALE, V_SCALE = 0.0171, 0.0157


def fp8_values():
    """The 256 E4M3 values as FP64."""
    import torch
    return torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()


class Case:
    """A cache, a table and query rows.  `rows` None: the one-row form."""

    def __init__(self, seed, lens, rows, hq, hkv, window, sinks, page=16, layout="NHD",
                 dtype="bf16", spare=3, freed=False):
        rng = np.random.default_rng(seed)
        self.lens, self.hq, self.hkv, self.page = list(lens), hq, hkv, page
        self.layout, self.dtype, self.window, self.sinks = layout, dtype, window, sinks
        self.single = rows is None
        self.rows = [1] * len(lens) if rows is None else list(rows)
        self.pool, self.indptr, self.indices, self.last = mx.table(rng, lens, page, spare)
        if freed:  # pages that no row sees: given away
            for r, (n, m) in enumerate(zip(self.lens, self.rows)):
                first = max(0, n - m + 1 - window) if window else 0
                self.indices[self.indptr[r] + -(-sinks // page):
                             self.indptr[r] + first // page] = -1
        shape = (self.pool, hkv, page)
        if dtype == "mxfp4":
            self.cache = [mx.random_cache(rng, self.pool, page, hkv) for _ in "kv"]
        elif dtype == "fp8_e4m3":
            table = fp8_values()
            codes = np.flatnonzero(np.abs(table) <= 240).astype(np.uint8)
            self.cache = [codes[rng.integers(0, len(codes), (*shape, D))] for _ in "kv"]
        else:
            self.cache = [mx.bf16_round(rng.standard_normal((*shape, D))) for _ in "kv"]
        self.nnz = sum(self.rows)
        self.q = mx.bf16_round(rng.standard_normal((max(1, self.nnz), hq, D)))

    # ---- the definition -----------------------------------------------------------
    def values(self, which):
        """FP64 [pool, hkv, page, 128] of K (0) or V (1)."""
        c = self.cache[which]
        if self.dtype == "mxfp4":
            return mx.values(*c)
        if self.dtype == "fp8_e4m3":
            return fp8_values()[c] * float(np.float32((K_SCALE, V_SCALE)[which]))
        return c

    def reference(self):
        """O [nnz, hq, 128], LSE [nnz, hq], A (as O) and S [nnz, hq] of the module's text."""
        kv = [self.values(0), self.values(1)]
        o, a = np.zeros((self.nnz, self.hq, D)), np.zeros((self.nnz, self.hq, D))
        lse, s_abs = np.zeros((self.nnz, self.hq)), np.zeros((self.nnz, self.hq))
        at, group = 0, self.hq // self.hkv
        for r, (n, m) in enumerate(zip(self.lens, self.rows)):
            if m == 0:
                continue
            t = np.arange(n)
            p = np.arange(n - m, n)[:, None]
            seen = t <= p
            if self.window:
                seen &= (t > p - self.window) | (t < self.sinks)
            used = np.flatnonzero(seen.any(0))
            slots = self.indices[self.indptr[r] + used // self.page], used % self.page
            for h in range(self.hkv):
                k, v = (c[slots[0], h, slots[1]] for c in kv)
                for g in range(h * group, (h + 1) * group):
                    q = self.q[at:at + m, g]
                    with np.errstate(invalid="ignore", over="ignore"):
                        s = np.where(seen[:, used], q @ k.T * D ** -0.5, -np.inf)
                        top = s.max(1, keepdims=True)
                        w = np.exp(s - top)
                        total = w.sum(1, keepdims=True)
                        if np.isfinite(v).all():
                            o[at:at + m, g] = w / total @ v
                        else:  # (a weight of zero times an infinity)
                            o[at:at + m, g] = np.stack([
                                (w[i, w[i] != 0] / total[i]) @ v[w[i] != 0] for i in range(m)])
                        a[at:at + m, g] = w / total @ np.abs(np.where(np.isfinite(v), v, 0))
                        lse[at:at + m, g] = ((top + np.log(total)) * LOG2E)[:, 0]
                        sa = np.where(seen[:, used], np.abs(q) @ np.abs(k).T, 0)
                        s_abs[at:at + m, g] = np.nanmax(sa, 1) * D ** -0.5 * LOG2E
            at += m
        return o, lse, a, s_abs

    def check(self, out, lse, long_tile=False, only=None):
        """`only`: the query rows that are compared."""
        o, l, a, s = (x[slice(None) if only is None else only] for x in self.reference())
        out, lse = (x[slice(None) if only is None else only] for x in (out, lse))
        n = max(self.lens)
        score = 128 * 2.0 ** -24 * s
        weight = 2 * 0.6932 * score[..., None] + (2.0 ** -7 if long_tile else 2.0 ** -14) \
            + n * 2.0 ** -23 + 2.0 ** -20
        tol = 2.0 ** -8 * np.abs(o) + weight * a + 1e-30
        tol_l = score + 2.0 ** -14 + n * 2.0 ** -23 + np.abs(l) * 2.0 ** -21
        e, el = np.abs(out - o) / tol, np.abs(lse - l) / tol_l
        assert e.max() <= 1, f"O off by {e.max():.3g} of its bound at {np.unravel_index(e.argmax(), e.shape)}"
        assert el.max() <= 1, f"LSE off by {el.max():.3g} of its bound at {np.unravel_index(el.argmax(), el.shape)}"

    # ---- the library ----------------------------------------------------------------
    def operands(self, torch, offset=0):
        """Device operands by name; `offset` bytes past an aligned start."""
        def put(x):
            b = torch.empty(x.nbytes + 16, dtype=torch.uint8, device="cuda")
            w = b[offset:offset + x.nbytes]
            w.copy_(torch.from_numpy(np.ascontiguousarray(x).view(np.uint8).reshape(-1)).cuda())
            return w

        def paged(x):
            return x if self.layout == "HND" else np.ascontiguousarray(x.swapaxes(1, 2))

        def ints(x):
            return torch.from_numpy(np.ascontiguousarray(np.asarray(x, np.int32))).cuda()

        def bf16(x):
            return put(mx.bf16_bits(x)).view(torch.bfloat16)

        d = {"q": bf16(self.q[:self.nnz]), "indptr": ints(self.indptr),
             "indices": ints(self.indices), "last": ints(self.last)}
        if not self.single:
            d["qo"] = ints(np.concatenate([[0], np.cumsum(self.rows)]))
        for name, c in zip("kv", self.cache):
            if self.dtype == "mxfp4":
                d[name] = put(paged(c[0]))
                d[name + "_mx"] = put(c[1])
            else:
                d[name] = put(paged(c)) if self.dtype == "fp8_e4m3" else bf16(paged(c))
        if self.dtype == "fp8_e4m3":
            d["kv_scales"] = torch.tensor([K_SCALE, V_SCALE], device="cuda")
        return d

    def spec(self, L, **other):
        form = dict(window=self.window, sinks=self.sinks, explicit_rows=not self.single,
                    kv_layout=self.layout, kv_dtype=self.dtype, kv_page_size=self.page)
        return L.WindowPagedAttentionSpec(self.nnz, len(self.lens), self.pool, self.hq, self.hkv,
                                          **(form | other))

    def plan(self, L, tile_cols=0, capacity=False, **other):
        spec = self.spec(L, **other)
        if self.single:
            return L.DecodeProvider.load(0).plan_window_paged_batch(spec, indices_capacity=capacity)
        return L.PrefillProvider.load(0).plan_window_paged(spec, indices_capacity=capacity,
                                                           tile_cols=tile_cols)

    def args(self, L, bindings, d, out, lse):
        r = {k: bindings.bind_read(v) for k, v in d.items()}
        return L.WindowPagedAttentionArgs(
            r["q"], r["k"], r["v"], r["indptr"], r["indices"], r["last"],
            bindings.bind_read_write(out).write(), bindings.bind_read_write(lse).write(),
            qo_indptr=r.get("qo"), kv_scales=r.get("kv_scales"), key_scales=r.get("k_mx"),
            value_scales=r.get("v_mx"))

    def outputs(self, torch):
        return (torch.full((self.nnz, self.hq, D), 7.0, dtype=torch.bfloat16, device="cuda"),
                torch.full((self.nnz, self.hq), 7.0, device="cuda"))

    def run(self, torch, L, d=None, offset=0, stream=None, **plan):
        """(O, LSE) in FP64, after one command."""
        d = d or self.operands(torch, offset)
        out, lse = self.outputs(torch)
        torch.cuda.synchronize()
        queue = L.CommandQueue(stream or torch.cuda.current_stream(), 1)
        b = queue.bindings(16)
        p = self.plan(L, **plan)
        a = self.args(L, b, d, out, lse)
        scope = queue.begin(b)
        p.enqueue_into(scope, a)
        scope.finish().wait()
        return host(out), host(lse)


def host(t):
    import torch
    if t.dtype == torch.bfloat16:
        return mx.bf16_values(t.view(torch.int16).cpu().numpy().view(np.uint16))
    return t.cpu().numpy().astype(np.float64)
