"""The paged key-value cache on the GPU: the append and the attention over it
against the oracle's float64 restatement (oracle/kv.py).

Bars. u = 2^-24, half a step of f32.
 * Append: a normed head element carries three roundings (the factor, two
   products), a rotated pair two products, a sum and the angle's own error (a
   cosine of an angle rounded to f32 turns: pi u, its evaluation 2u), so
   |y - ref| <= 16 u (|a| + |b|), plus half a step of the cache's type.
 * Attention, each output: scores are sums of dk products of up to 24 bits, with
   A = max sum |scale q k|: off by (dk + 8) u A (rounded operands, sums, the
   change of base); that moves an average of the values by at most twice as
   much times max|v|. Sums over n keys: chains of at most n / 8 + 300 additions.
   |y - ref| <= u max|v| (2 (dk + 8) A + n / 8 + 300), a bound for the worst case.
 * Attention, all outputs together: roundings are independent, so of a sum of
   terms about their square root remains; operands of 22 bits leave 2^-22 of a
   score of order 1, which is of the order of the output's relative error.
   norm(y - ref) <= 2^-19 norm(ref): eight times that. It is two hundred
   times below what one rounding to 16 bits would leave.
"""
import threading

import numpy as np
import pytest

import kv as O
import mynah_hip as M

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
TYPES = {"f32": M.F32, "f16": M.F16, "bf16": M.BF16}


def say(*a):
    print(*a, flush=True)


def torch_type(t):
    import torch
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[t]


def f64(t):
    return t.double().cpu().numpy()


class Case:
    """A cache with random contents and a batch over it: `new` and `length` per sequence."""

    def __init__(self, typ, dk, heads, kv_heads, page, new, length, seed=0, pad=0, spare=2, ldx=0, max_len=None,
                 max_new=None, sigma=1.0):
        import torch
        self.typ, self.dk, self.heads, self.kv_heads, self.page = typ, dk, heads, kv_heads, page
        g = torch.Generator().manual_seed(seed + 1)
        need = [-(-max(n, 0) // page) for n in length]
        self.n_pages = sum(need) + spare
        order = torch.randperm(self.n_pages, generator=g).int()
        most = max(need + [1])
        self.pages = torch.full((len(length), most), -1, dtype=torch.int32)
        at = 0
        for b, n in enumerate(need):
            self.pages[b, :n] = order[at:at + n]
            at += n
        self.starts = [0]
        for n in new:
            self.starts.append(self.starts[-1] + n)
        self.real = self.starts[-1]
        self.rows = self.real + pad
        self.length = list(length)
        self.max_new = max(list(new) + [1]) if max_new is None else max_new
        self.max_len = max(list(length) + [1]) if max_len is None else max_len
        rnd = lambda *s: torch.randn(*s, generator=g)   # noqa: E731
        self.k_pool = rnd(self.n_pages, kv_heads, page, dk).to(torch_type(typ)).cuda()
        self.v_pool = rnd(self.n_pages, kv_heads, page, dk).to(torch_type(typ)).cuda()
        self.ldq = heads * dk + ldx
        self.q = (rnd(self.rows, self.ldq) * sigma).cuda()
        self.ldk = kv_heads * dk + ldx
        self.k, self.v = rnd(self.rows, self.ldk).cuda(), rnd(self.rows, self.ldk).cuda()
        self.upload()

    def upload(self):
        import torch
        self.d_start = torch.tensor(self.starts, dtype=torch.int32).cuda()
        self.d_len = torch.tensor(self.length, dtype=torch.int32).cuda()
        self.d_pages = self.pages.cuda()
        self.cache = M.kv_cache(TYPES[self.typ], self.k_pool.data_ptr(), self.v_pool.data_ptr(), self.n_pages, self.page,
                                self.kv_heads, self.dk)
        self.batch = M.kv_batch(self.d_start.data_ptr(), self.d_len.data_ptr(), self.d_pages.data_ptr(),
                                len(self.length), self.rows, self.pages.shape[1], self.max_new, self.max_len)

    def heads_of(self, x, n):
        return x[:, :n * self.dk].reshape(self.rows, n, self.dk)

    def attend(self, gpu, scale=None, causal=1, window=0, sinks=0, out=None, stream=0, **kw):
        import torch
        scale = self.dk ** -0.5 if scale is None else scale
        if out is None:
            out = torch.full((self.rows, self.ldq), 7.25, device="cuda")
        torch.cuda.synchronize()
        M.kv_attention_dev(gpu, self.cache, self.batch, self.q.data_ptr(), self.ldq, self.heads, out.data_ptr(), self.ldq,
                           scale, causal, window, sinks, stream=stream, **kw)
        torch.cuda.synchronize()
        return out

    def check(self, gpu, scale=None, causal=1, window=0, sinks=0):
        scale = self.dk ** -0.5 if scale is None else scale
        out = self.attend(gpu, scale, causal, window, sinks)
        assert (out[self.real:] == 7.25).all() and (out[:, self.heads * self.dk:] == 7.25).all()
        y = f64(self.heads_of(out, self.heads))[:self.real]
        ref, terms, count, vmax = (x[:self.real] for x in O.attention(
            f64(self.k_pool), f64(self.v_pool), self.starts, self.length, self.pages.numpy(),
            f64(self.heads_of(self.q, self.heads)), float(np.float32(scale)), causal, window, sinks, self.max_len))
        lim = U * vmax * (2 * (self.dk + 8) * terms + count / 8 + 300)
        err = np.abs(y - ref)
        assert np.isfinite(y).all()
        worst = (err.max(-1) / np.maximum(lim, 1e-300)).max() if err.any() else 0.0
        rel = np.linalg.norm(y - ref) / max(np.linalg.norm(ref), 1e-300)
        say(f"  worst {worst:.3g} of the bound, norm {rel:.3g}")
        assert (err <= lim[..., None]).all()
        assert rel <= 2.0 ** -19 * max(1.0, terms.max(initial=0.0) / 8)
        return out


# --------------------------------------------------------------------- append
def expect_append(c, prep, got_q, q_in, k_in, v_in, k_pool, v_pool):
    eps = float(np.float32(prep.get("eps", 0.0)))
    kw = dict(q_norm=prep.get("qn"), k_norm=prep.get("kn"), eps=eps, rot=prep.get("rot", 0),
              interleaved=prep.get("interleaved", False), freq=prep.get("freq"))
    ref = O.append(f64(k_pool), f64(v_pool), c.starts, c.length, c.pages.numpy(), q_in, k_in, v_in, **kw)
    # the size of what a pair is made of: the same without rotation, both members
    flat = O.append(f64(k_pool), f64(v_pool), c.starts, c.length, c.pages.numpy(), q_in, k_in, v_in,
                    q_norm=prep.get("qn"), k_norm=prep.get("kn"), eps=eps)
    rot, dk = kw["rot"], c.dk
    mate = np.arange(dk)
    if kw["interleaved"]:
        mate[:rot] ^= 1
    else:
        mate[:rot] = (mate[:rot] + rot // 2) % max(rot, 1)
    size = [np.abs(f) + np.abs(f[..., mate]) for f in flat]
    half, tiny = {"f32": (0.0, 0.0), "f16": (2.0 ** -11, 2.0 ** -25), "bf16": (2.0 ** -8, 0.0)}[c.typ]
    y = f64(c.heads_of(got_q, c.heads))[:c.real]
    assert (np.abs(y - ref[0][:c.real]) <= 16 * U * size[0][:c.real]).all()
    for got, r, s, before in ((c.k_pool, ref[1], size[1], k_pool), (c.v_pool, ref[2], None, v_pool)):
        g = f64(got)
        lim = (16 * U * s if s is not None else 0.0) + half * np.abs(r) * (1 + 32 * U) + tiny
        assert (np.abs(g - r) <= lim).all()
        untouched = r == f64(before)      # slots that no row's position names
        assert (g[untouched] == f64(before)[untouched]).all()


def run_append(gpu, c, prep, in_place=False, with_q=True):
    import torch
    q0, k0, v0 = c.q.clone(), c.k_pool.clone(), c.v_pool.clone()
    out = c.q if in_place else torch.full_like(c.q, 7.25)
    dev = {n: torch.from_numpy(np.asarray(prep[n])).cuda() for n in ("qn", "kn", "freq") if prep.get(n) is not None}
    p = M.kv_prep(q_norm=dev["qn"].data_ptr() if "qn" in dev else None,
                  k_norm=dev["kn"].data_ptr() if "kn" in dev else None, eps=prep.get("eps", 0.0),
                  rot=prep.get("rot", 0), interleaved=prep.get("interleaved", False),
                  freq=dev["freq"].data_ptr() if "freq" in dev else None)
    torch.cuda.synchronize()
    M.kv_append_dev(gpu, c.cache, c.batch, p if prep else None, c.q.data_ptr() if with_q else None, c.ldq,
                    c.heads if with_q else 0, out.data_ptr() if with_q else None, c.ldq, c.k.data_ptr(), c.ldk,
                    c.v.data_ptr(), c.ldk)
    torch.cuda.synchronize()
    if with_q:
        keep = q0 if in_place else torch.full_like(q0, 7.25)
        assert (out[c.real:] == keep[c.real:]).all()
        assert (out[:, c.heads * c.dk:] == keep[:, c.heads * c.dk:]).all()
    else:
        out = c.q
    expect_append(c, prep, out, f64(c.heads_of(q0, c.heads)), f64(c.heads_of(c.k, c.kv_heads)),
                  f64(c.heads_of(c.v, c.kv_heads)), k0, v0)


def preps(dk, seed=3):
    r = np.random.default_rng(seed)
    w = lambda: (1 + 0.2 * r.standard_normal(dk)).astype(np.float32)   # noqa: E731
    f = lambda rot: 10000.0 ** (-np.arange(0, rot, 2) / rot)           # noqa: E731
    return {"plain": {}, "norm": dict(qn=w(), kn=w(), eps=1e-6), "rot": dict(rot=dk, freq=f(dk)),
            "both": dict(qn=w(), kn=w(), eps=1e-5, rot=dk, freq=f(dk)),
            "part": dict(kn=w(), eps=1e-6, rot=dk // 2, freq=f(dk // 2)),
            "inter": dict(qn=w(), kn=w(), eps=1e-6, rot=dk, interleaved=True, freq=f(dk)),
            "inter8": dict(rot=8, interleaved=True, freq=f(8))}


@pytest.mark.parametrize("prep", ["plain", "norm", "rot", "both", "part", "inter", "inter8"])
@pytest.mark.parametrize("typ,dk", [("f32", 128), ("f16", 128), ("bf16", 128), ("f32", 64), ("f16", 64), ("bf16", 64)])
def test_append(gpu, typ, dk, prep):
    """Ragged new rows on top of cached ones, odd pages, rows behind the last sequence, strided rows."""
    say("append", typ, dk, prep)
    c = Case(typ, dk, 6, 2, 7, [3, 0, 1, 12], [10, 5, 1, 12], pad=3, ldx=8)
    run_append(gpu, c, preps(dk)[prep])


@pytest.mark.parametrize("heads,kv_heads,page,new,length", [
    (1, 1, 1, [1], [1]), (8, 8, 16, [1] * 5, [1, 16, 17, 400, 33]), (71, 1, 64, [2, 5], [64, 70]),
    (32, 8, 25, [40], [40]), (3, 3, 5, [0, 0, 4, 0], [9, 0, 4, 2])])
def test_append_shapes(gpu, heads, kv_heads, page, new, length):
    say("append shapes", heads, kv_heads, page, new, length)
    c = Case("f16", 128, heads, kv_heads, page, new, length, pad=1)
    run_append(gpu, c, preps(128)["both"])


@pytest.mark.parametrize("nseq", [255, 256, 257, 1500])
def test_append_many_sequences(gpu, nseq):
    """The search for a row's sequence: empty ones among them, at both ends too."""
    say("append many sequences", nseq)
    r = np.random.default_rng(nseq)
    new = [int(x) for x in r.integers(0, 3, nseq)]
    new[0] = new[-1] = 0
    length = [n + int(o) for n, o in zip(new, r.integers(0, 20, nseq))]
    run_append(gpu, Case("bf16", 64, 2, 1, 4, new, length, pad=2), preps(64)["both"])


def test_append_in_place_and_without_q(gpu):
    for how in (dict(in_place=True), dict(with_q=False)):
        say("append", how)
        prep = preps(128)["both"] if "in_place" in how else {k: v for k, v in preps(128)["part"].items()}
        c = Case("f32", 128, 4, 4, 16, [3, 9], [30, 9], ldx=4)
        if "with_q" in how:
            prep = {}   # (expect_append then compares q with itself)
        run_append(gpu, c, prep, **how)


def test_append_far_positions(gpu):
    """Angles at positions near 2^20 and 2^30: formed in 64 bits."""
    import torch
    for pos in (1 << 20, (1 << 30) - 8):
        say("append far", pos)
        c = Case("f32", 128, 2, 1, 64, [3], [3])
        c.length = [pos]
        c.pages = torch.full((1, (pos >> 6) + 1), -1, dtype=torch.int32)
        c.pages[0, (pos - 1) >> 6] = 1
        c.upload()
        run_append(gpu, c, preps(128)["rot"])


def test_append_bad_tables(gpu):
    """Pages outside the pool, keys past the table, fewer keys than rows: nothing of those is written."""
    import torch
    for length, row in (([9, 12], [0, 9]), ([9, 12], [-1, 1]), ([9, 30], [0, 1]), ([2, 8], [0, 1]), ([-5, 2 ** 30], [0, 1])):
        say("append bad tables", length, row)
        c = Case("f16", 64, 2, 2, 4, [5, 4], [9, 12], pad=1)
        c.length = length
        if row != [0, 1]:
            c.pages[0, 1], c.pages[1, 2] = (c.n_pages, -7) if row[1] == 9 else (2 ** 31 - 1, -2 ** 31)
        c.upload()
        run_append(gpu, c, preps(64)["rot"])
    # rows that row_start gives to no sequence, or that it does not have
    c = Case("f16", 64, 2, 2, 4, [5, 4], [9, 12])
    before = c.k_pool.clone()
    for starts in ([9, 9, 9], [2, 2, 2], [0, 0, 0], [-3, -3, -2]):
        c.starts = starts
        c.upload()
        out = torch.full_like(c.q, 7.25)
        torch.cuda.synchronize()
        M.kv_append_dev(gpu, c.cache, c.batch, None, c.q.data_ptr(), c.ldq, 2, out.data_ptr(), c.ldq, c.k.data_ptr(),
                        c.ldk, c.v.data_ptr(), c.ldk)
        torch.cuda.synchronize()
        assert (out == 7.25).all() and torch.equal(before, c.k_pool)


def test_append_special_values(gpu):
    """Infinity past f16's range, ties to even, NaN as NaN, and rows beside them untouched by it."""
    import torch
    c = Case("f16", 64, 2, 1, 4, [4], [4])
    c.k[0, :4] = torch.tensor([70000.0, -65520.0, 65519.0, float("nan")])
    c.k[1, :4] = torch.tensor([1 + 2.0 ** -11, 1 + 3 * 2.0 ** -11, 2.0 ** -25, 3 * 2.0 ** -25])
    c.q[2, 5] = float("inf")
    torch.cuda.synchronize()
    out = torch.empty_like(c.q)
    M.kv_append_dev(gpu, c.cache, c.batch, None, c.q.data_ptr(), c.ldq, 2, out.data_ptr(), c.ldq, c.k.data_ptr(), c.ldk,
                    c.v.data_ptr(), c.ldk)
    torch.cuda.synchronize()
    assert torch.equal(out, c.q)
    pg = int(c.pages[0, 0])
    assert torch.equal(c.k_pool[pg, 0].isnan(), c.k.half().isnan())
    assert torch.equal(c.k_pool[pg, 0].nan_to_num(1.5), c.k.half().nan_to_num(1.5))
    assert torch.equal(c.v_pool[pg, 0], c.v.half())


# ------------------------------------------------------------------ attention
STEP = [1, 15, 16, 17, 63, 64, 65, 255, 256, 257, 300]


@pytest.mark.parametrize("typ,dk", [("f32", 128), ("f16", 128), ("bf16", 128), ("f32", 64), ("f16", 64), ("bf16", 64)])
@pytest.mark.parametrize("heads,kv_heads,page", [(2, 2, 16), (8, 2, 64), (5, 1, 7)])
def test_step(gpu, typ, dk, heads, kv_heads, page):
    """One new row a sequence; lengths around every block's and chunk's end."""
    say("step", typ, dk, heads, kv_heads, page)
    Case(typ, dk, heads, kv_heads, page, [1] * len(STEP), STEP, pad=2, ldx=4).check(gpu)


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads", [(16, 1), (17, 1), (71, 1), (7, 1), (6, 2)])
def test_step_head_groups(gpu, typ, heads, kv_heads):
    say("step groups", typ, heads, kv_heads)
    Case(typ, 64, heads, kv_heads, 16, [1] * 3, [40, 270, 600]).check(gpu)


@pytest.mark.parametrize("typ,dk", [("f32", 64), ("f16", 128), ("bf16", 128)])
@pytest.mark.parametrize("window,sinks", [(1, 0), (5, 2), (64, 4), (100, 0), (257, 70), (300, 64), (5000, 3)])
def test_step_window(gpu, typ, dk, window, sinks):
    say("step window", typ, dk, window, sinks)
    Case(typ, dk, 4, 2, 16, [1] * 7, [1, 5, 64, 131, 400, 801, 1500]).check(gpu, window=window, sinks=sinks)


@pytest.mark.parametrize("typ,dk", [("f32", 128), ("f16", 128), ("bf16", 64)])
@pytest.mark.parametrize("new,length", [([2, 4, 1], [2, 70, 300]), ([8, 3], [1000, 3]), ([17, 33, 0, 1], [17, 64, 9, 130]),
                                        ([64], [64]), ([65], [65]), ([130, 7], [200, 400])])
@pytest.mark.parametrize("window,sinks", [(0, 0), (40, 3)])
def test_several_rows(gpu, typ, dk, new, length, window, sinks):
    """A few new rows, and prompts, in causal order, with and without a window."""
    say("rows", typ, dk, new, length, window, sinks)
    Case(typ, dk, 6, 2, 25, new, length, pad=5).check(gpu, window=window, sinks=sinks)


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,dk", [(4, 4, 64), (8, 1, 64), (8, 2, 128), (3, 1, 128)])
def test_prompt(gpu, typ, heads, kv_heads, dk):
    say("prompt", typ, heads, kv_heads, dk)
    Case(typ, dk, heads, kv_heads, 16, [300, 129], [300, 420], pad=9, ldx=8).check(gpu)


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("window,sinks", [(1, 0), (3, 1), (64, 4), (90, 65), (200, 0), (150, 130)])
def test_prompt_window(gpu, typ, window, sinks):
    say("prompt window", typ, window, sinks)
    Case(typ, 64, 4, 2, 16, [350, 40], [350, 460]).check(gpu, window=window, sinks=sinks)


@pytest.mark.parametrize("nseq", [2, 63, 64, 65, 256, 257, 600])
@pytest.mark.parametrize("typ", ["f16", "f32"])
def test_prompts_of_many_sequences(gpu, typ, nseq):
    """The order in which prompts' tiles are taken: sequences of no row, of one tile, of several."""
    say("many prompts", typ, nseq)
    r = np.random.default_rng(nseq)
    new = [int(x) for x in r.choice([0, 1, 5, 16, 17, 40], nseq)]
    new[-1] = 0
    new[nseq // 2] = 33
    c = Case(typ, 64, 8, 1, 16, new, [n + int(o) for n, o in zip(new, r.integers(0, 9, nseq))], pad=3)
    c.check(gpu)


@pytest.mark.parametrize("typ,dk", [("f32", 128), ("f16", 128), ("bf16", 128), ("f32", 64), ("f16", 64), ("bf16", 64)])
@pytest.mark.parametrize("new,old,window,sinks", [(40, 9000, 0, 0), (9, 9000, 0, 0), (130, 3000, 0, 0), (130, 3000, 700, 5)])
def test_parts_of_long_prompts(gpu, typ, dk, new, old, window, sinks):
    """New rows on long caches, split over the keys and joined, against the definition on the GPU in 64 bits."""
    import torch
    say("part", typ, dk, new, old, window)
    n = new + old
    c = Case(typ, dk, 6, 2, 48, [new], [n])
    out = c.attend(gpu, window=window, sinks=sinks).view(new, 6, dk).double()
    flat = lambda p: p[c.d_pages[0].long()].permute(1, 0, 2, 3).reshape(2, -1, dk)[:, :n].double()   # noqa: E731
    k, v = flat(c.k_pool), flat(c.v_pool)
    p = torch.arange(old, n, device="cuda")[:, None]
    j = torch.arange(n, device="cuda")[None]
    see = (j <= p) & ((j > p - window) | (j < sinks)) if window else j <= p
    for h in range(6):
        s = (c.q.view(new, 6, dk)[:, h].double() @ k[h // 3].T.contiguous() * dk ** -0.5).masked_fill(~see, -np.inf)
        ref = torch.softmax(s, 1) @ v[h // 3]
        assert ((out[:, h] - ref).norm() / ref.norm()).item() <= 2.0 ** -19


@pytest.mark.parametrize("typ,dk", [("f32", 128), ("f16", 64), ("bf16", 128)])
@pytest.mark.parametrize("new", [[1, 1], [4, 4], [40, 3], [70, 3]])
def test_not_causal(gpu, typ, dk, new):
    say("not causal", typ, dk, new)
    Case(typ, dk, 4, 4, 25, new, [200, 75]).check(gpu, causal=0)


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
def test_rows_that_see_nothing(gpu, typ):
    """Empty caches, fewer keys than rows, negative lengths: zeros, and rows that see something are right."""
    say("see nothing", typ)
    for new, length in (([1, 1], [0, 3]), ([5, 2], [3, 0]), ([80, 3], [40, 3])):
        c = Case(typ, 64, 4, 2, 16, new, [max(x, 1) for x in length])
        c.length = length
        c.upload()
        out = c.check(gpu)
        assert (out[0, :4 * 64] == 0).all()
    c.length = [-7, -2 ** 31]
    c.upload()
    assert (c.attend(gpu, causal=0)[:, :4 * 64] == 0).all()


@pytest.mark.parametrize("new", [[1, 1, 1], [3, 2, 1], [90, 20, 70]])
def test_bounds_hold(gpu, new):
    """max_len hides what lies past it, max_new leaves rows as they are; pages outside the pool are not seen."""
    say("bounds", new)
    length = [n + o for n, o in zip(new, (100, 0, 400))]
    c = Case("f16", 64, 4, 2, 16, new, length, max_len=150)
    c.check(gpu)
    c = Case("f16", 64, 4, 2, 16, new, length)
    c.pages[0, 0], c.pages[0, 3], c.pages[2, 5], c.pages[2, 11] = c.n_pages, -1, 2 ** 31 - 1, -2 ** 31
    c.pages[1, 0] = c.n_pages + 1
    c.upload()
    out = c.check(gpu)
    assert (out[c.starts[1], :256] == 0).all()
    if max(new) > 1:
        c = Case("f16", 64, 4, 2, 16, new, length)
        whole = c.attend(gpu)
        c.max_new = 2
        c.upload()
        out = c.attend(gpu)
        for b, n in enumerate(new):
            assert (out[c.starts[b] + min(n, 2):c.starts[b + 1]] == 7.25).all()
            a, z = out[c.starts[b]:c.starts[b] + min(n, 2)], whole[c.starts[b]:c.starts[b] + min(n, 2)]
            assert (a - z).abs().max() <= 1e-4


@pytest.mark.parametrize("new", [[1, 1], [4, 3], [40, 70]])
def test_more_keys_than_the_table_holds(gpu, new):
    """len past max_pages * page_size, under max_len: the keys that the table has no page for are not seen."""
    say("past the table", new)
    c = Case("bf16", 64, 4, 2, 16, new, [n + 100 for n in new], max_len=1 << 20)
    held = c.pages.shape[1] * 16
    for length in ([held + 1, held], [held + 3, held + 900], [10 ** 6, 2 ** 30]):
        c.length = length
        c.pages[c.pages < 0] = 0
        c.upload()
        c.max_len = held       # (the oracle's list of keys; the call still has 2^20)
        c.check(gpu)
        c.max_len = 1 << 20


@pytest.mark.parametrize("new", [[1, 1], [4, 3], [40, 70]])
def test_rows_before_the_first(gpu, new):
    """row_start that begins behind the buffers' first rows: those are left as they are."""
    import torch
    say("rows before the first", new)
    c = Case("f16", 64, 4, 2, 16, new, [n + 50 for n in new], pad=3)
    ref = c.attend(gpu)
    q, k = c.q.clone(), c.k.clone()
    c.q[3:], c.k[3:] = q[:-3], k[:-3]
    c.starts = [x + 3 for x in c.starts]
    c.upload()
    out = c.attend(gpu)
    assert (out[:3] == 7.25).all() and torch.equal(out[3:], ref[:-3])
    got = torch.full_like(c.q, 7.25)
    torch.cuda.synchronize()
    M.kv_append_dev(gpu, c.cache, c.batch, None, c.q.data_ptr(), c.ldq, 4, got.data_ptr(), c.ldq, c.k.data_ptr(), c.ldk,
                    c.v.data_ptr(), c.ldk)
    torch.cuda.synchronize()
    assert (got[:3] == 7.25).all() and torch.equal(got[3:], c.q[3:])


def test_row_start_of_no_use(gpu):
    c = Case("bf16", 64, 4, 2, 16, [5, 4], [9, 120])
    for starts in ([9, 9, 9], [0, 0, 0], [-3, -3, -2], [5, 5, 5]):
        c.starts = starts
        c.upload()
        assert (c.attend(gpu) == 7.25).all()


@pytest.mark.parametrize("new", [[5, 4], [40, 30], [1] * 70])
def test_row_start_at_the_ends_of_its_type(gpu, new):
    """2^31 - 1 before -2^31, whose difference is 1 in 32 bits, and the like: rows of no sequence stay as they are."""
    import torch
    low, high = -2 ** 31, 2 ** 31 - 1
    n = len(new) + 1
    c = Case("f16", 64, 4, 2, 16, new, [x + 70 for x in new])
    before = c.k_pool.clone()
    for first, rest in ((high, low), (high, low + 3), (high - 1, low), (low, low), (high, high), (c.rows, low)):
        say("row_start", new, first, rest)
        c.starts = [first] + [rest] * (n - 1)
        c.upload()
        assert (c.attend(gpu) == 7.25).all()
        out = torch.full_like(c.q, 7.25)
        torch.cuda.synchronize()
        M.kv_append_dev(gpu, c.cache, c.batch, None, c.q.data_ptr(), c.ldq, 4, out.data_ptr(), c.ldq, c.k.data_ptr(),
                        c.ldk, c.v.data_ptr(), c.ldk)
        torch.cuda.synchronize()
        assert (out == 7.25).all() and torch.equal(before, c.k_pool)


SPECIAL = [float("nan"), float("inf"), -float("inf")]


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("new,window", [([1, 1], 0), ([1, 1], 50), ([3, 2], 0), ([3, 2], 50), ([9, 12], 0), ([16, 3], 50),
                                        ([90, 75], 0), ([90, 75], 50)])
def test_what_is_not_seen_changes_nothing(gpu, typ, new, window):
    """Slots behind a sequence's end, in its last page and in pages of no sequence: NaN and infinities there leave every
    bit as it was; so do huge finite ones."""
    import torch
    say("not seen", typ, new, window)
    length = [n + o for n, o in zip(new, (70, 200))]
    c = Case(typ, 64, 4, 2, 16, new, length)
    base = c.attend(gpu, window=window, sinks=3 if window else 0)
    seen = torch.zeros(c.n_pages, 16, dtype=torch.bool)
    for b, n in enumerate(length):
        first = n - new[b] - window + 1 if window else 0
        for j in range(n):
            if j >= first or j < 3:
                seen[int(c.pages[b, j // 16]), j % 16] = True
    hidden = (~seen).cuda()[:, None, :, None].expand_as(c.k_pool)
    for bad in SPECIAL + [3e4]:
        c.k_pool[hidden] = bad
        c.v_pool[hidden] = bad
        assert torch.equal(c.attend(gpu, window=window, sinks=3 if window else 0), base), bad


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("new", [3, 10, 100])
@pytest.mark.parametrize("where", ["k", "v"])
def test_only_rows_that_see_a_nan_have_it(gpu, typ, new, where):
    """A NaN (or infinity) in one key or value of a sequence's new rows: earlier rows, and later ones whose window it has
    left, keep every bit; the others are not finite (in that feature, for a value)."""
    import torch
    for window in (0, 2, 40):
        say("nan", typ, new, where, window)
        c = Case(typ, 64, 4, 2, 16, [new], [new + 30])
        base = c.attend(gpu, window=window)
        j = 30 + new // 2          # the key of row new // 2
        last = min(new, new // 2 + window) if window else new
        for bad in SPECIAL:
            pool = c.k_pool if where == "k" else c.v_pool
            keep = pool.clone()
            pool[int(c.pages[0, j // 16]), 1, j % 16, 5] = bad
            out = c.attend(gpu, window=window)
            pool.copy_(keep)
            a, z = out.view(c.rows, 4, 64), base.view(c.rows, 4, 64)
            assert torch.equal(a[:, :2], z[:, :2])                       # heads of the other K/V head
            assert torch.equal(a[:new // 2], z[:new // 2]) and torch.equal(a[last:], z[last:])
            if where == "v":
                assert not a[new // 2:last, 2:, 5].isfinite().any()
                rest = [f for f in range(64) if f != 5]
                assert torch.equal(a[new // 2:last, 2:][..., rest], z[new // 2:last, 2:][..., rest])
            elif bad != bad:
                assert a[new // 2:last, 2:].isnan().all()


@pytest.mark.parametrize("new", [1, 12, 70])
def test_special_queries(gpu, new):
    """A NaN in a head's q makes that head NaN and no other."""
    import torch
    c = Case("f16", 64, 4, 2, 16, [new, new], [new + 20, new + 3])
    base = c.attend(gpu)
    c.q[1, 70] = float("nan")
    out = c.attend(gpu).view(c.rows, 4, 64)
    assert out[1, 1].isnan().all()
    out[1, 1] = base.view(c.rows, 4, 64)[1, 1]
    assert torch.equal(out.view(c.rows, -1), base)


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("new", [1, 14, 80])
def test_scores_of_all_sizes(gpu, typ, new):
    """Scores that differ by hundreds (one key takes all), that are all alike, rows of q from 2^-40 to 2^30, zero rows."""
    import torch
    say("scores", typ, new)
    for sigma in (0.0, 1e-12, 20.0):
        Case(typ, 64, 4, 2, 16, [new, 1], [new + 200, 90], sigma=sigma).check(gpu)
    c = Case(typ, 64, 4, 2, 16, [new, 1], [new + 200, 90])
    c.q *= torch.exp2(torch.randint(-40, 6, (c.rows, 1), generator=torch.Generator().manual_seed(5)).float()).cuda()
    c.check(gpu)
    c.q[0] = torch.randn(c.q.shape[1], generator=torch.Generator().manual_seed(6)).cuda() * 2.0 ** 30
    c.check(gpu, scale=2.0 ** -31)
    c.check(gpu, scale=-2.0 ** -31)
    c.check(gpu, scale=0.0)
    # rows at the lower end of f32's range, subnormal ones among them: every score is 0 to f32, hidden keys stay hidden
    c.q[:] = torch.randn(c.q.shape, generator=torch.Generator().manual_seed(7)).cuda()
    c.q[0], c.q[-1] = c.q[0] * 2.0 ** -126 * 2.0 ** -16, c.q[-1] * 2.0 ** -124
    c.check(gpu)
    c.check(gpu, window=60, sinks=3)


def test_values_of_all_sizes(gpu):
    """Value features from 2^-24 to 2^15 (f16), 2^-100 to 2^100 (bf16, f32), each feature held to its own size."""
    import torch
    for typ, lo, hi in (("f16", -14, 12), ("bf16", -100, 100), ("f32", -100, 100), ("bf16", 0, 107), ("f32", 0, 107)):
        for new in (1, 12, 70):
            say("values", typ, new)
            c = Case(typ, 64, 4, 2, 16, [new], [new + 150])
            f = torch.exp2(torch.linspace(lo, hi, 64).round()).cuda()
            plain = c.attend(gpu)
            c.v_pool.copy_((c.v_pool.float() * f).to(c.v_pool.dtype))
            scaled = c.attend(gpu).view(c.rows, 4, 64) / f
            y, z = f64(scaled), f64(plain.view(c.rows, 4, 64))
            if typ != "f16":      # powers of two change no mantissa
                assert np.linalg.norm(y - z) <= 2.0 ** -20 * np.linalg.norm(z)
            else:                 # f16's subnormals round: half a step of 2^-24 at most, at 2^-14
                assert np.abs(y - z).max() <= 2.0 ** -10 + 2.0 ** -19 * np.abs(z).max()


@pytest.mark.parametrize("typ,heads,kv_heads", [("f16", 8, 1), ("bf16", 1, 1), ("f32", 4, 1)])
def test_long_cache(gpu, typ, heads, kv_heads):
    """Lengths on both sides of where chunks get longer, against the definition on the GPU in 64 bits."""
    import torch
    for n in (16383, 16385, 65536, 65537, 70001):
        say("long", typ, n)
        c = Case(typ, 64, heads, kv_heads, 32, [1], [n])
        out = c.attend(gpu).view(heads, 64).double()
        k = c.k_pool[c.d_pages[0].long()].permute(0, 2, 1, 3).reshape(-1, kv_heads, 64)[:n, 0].double()
        v = c.v_pool[c.d_pages[0].long()].permute(0, 2, 1, 3).reshape(-1, kv_heads, 64)[:n, 0].double()
        ref = torch.softmax(c.q.view(heads, 64).double() @ k.T.contiguous() / 8, 1) @ v
        rel = ((out - ref).norm() / ref.norm()).item()
        say(f"  {rel:.3g}")
        assert rel <= 2.0 ** -19


def test_pool_beyond_4_gib(gpu):
    """Keys and values behind the 2^32nd byte of their pools (and their 2^31st element)."""
    import torch
    n_pages = 2 ** 32 // (2 * 16 * 64 * 2) + 40      # 2 heads, pages of 16, f16
    say("pool pages", n_pages)
    for typ, pages in (("f16", n_pages), ("f32", n_pages)):
        c = Case(typ, 64, 4, 2, 16, [1, 2, 70], [100, 130, 200])
        big = [torch.empty(pages, 2, 16, 64, dtype=torch_type(typ), device="cuda") for _ in range(2)]
        far = pages - c.n_pages
        for x, small in zip(big, (c.k_pool, c.v_pool)):
            x[:c.n_pages] = float("nan")
            x[far:] = small
        ref = c.attend(gpu)
        small = c.k_pool, c.v_pool
        c.k_pool, c.v_pool, c.n_pages = big[0], big[1], pages
        c.pages = torch.where(c.pages >= 0, c.pages + far, c.pages)
        c.upload()
        assert torch.equal(c.attend(gpu), ref)
        M.kv_append_dev(gpu, c.cache, c.batch, None, None, 0, 0, None, 0, c.k.data_ptr(), c.ldk, c.v.data_ptr(), c.ldk)
        torch.cuda.synchronize()
        p = c.pages[2, 199 // 16]
        assert torch.equal(c.k_pool[p, :, 199 % 16].reshape(-1), c.k[-1].to(c.k_pool.dtype))
        assert torch.equal(c.v_pool[p, :, 199 % 16].reshape(-1), c.v[-1].to(c.k_pool.dtype))
        del big, small, c
        torch.cuda.empty_cache()


@pytest.mark.parametrize("new", [1, 4, 5, 8])
def test_same_bits_alone_and_in_a_batch(gpu, new):
    """A sequence's rows (up to 32 a K/V head) do not depend on the others of the call, nor a call on the ones before it."""
    import torch
    say("alone", new)
    lengths = [new + 3, new + 400, new + 1200]
    c = Case("f16", 128, 8, 2, 16, [new] * 3, lengths)
    whole = c.attend(gpu)
    assert torch.equal(c.attend(gpu), whole)
    starts, length, pages = c.starts, c.length, c.pages
    for b in range(3):
        c.starts, c.length, c.pages = starts[b:b + 2], length[b:b + 1], pages[b:b + 1]
        c.upload()
        out = c.attend(gpu)
        assert torch.equal(out[starts[b]:starts[b + 1]], whole[starts[b]:starts[b + 1]])


@pytest.mark.parametrize("new", [[1, 1], [3, 2], [200, 40]])
def test_out_in_place_of_q(gpu, new):
    import torch
    c = Case("bf16", 64, 8, 2, 16, new, [n + 900 for n in new])
    ref = c.attend(gpu)
    q = c.q.clone()
    out = c.attend(gpu, out=c.q)
    assert torch.equal(out[:c.real], ref[:c.real])
    c.q = q


def test_empty_calls(gpu):
    c = Case("f16", 64, 4, 2, 16, [1], [5])
    for f, v in (("nseq", 0), ("rows", 0), ("max_new", 0)):
        keep = getattr(c.batch, f)
        setattr(c.batch, f, v)
        assert (c.attend(gpu) == 7.25).all()
        setattr(c.batch, f, keep)
    c.batch.max_len = 0      # every key is past it
    assert (c.attend(gpu) == 0).all()
    # no rows, or no sequences either: buffers of no bytes have no address
    for b in (M.kv_batch(c.d_start.data_ptr(), c.d_len.data_ptr(), c.d_pages.data_ptr(), 1, 0, 1, 1, 16),
              M.kv_batch(None, None, None, 0, 0, 0, 0, 0)):
        M.kv_attention_dev(gpu, c.cache, b, None, c.ldq, 4, None, c.ldq, 0.125)
        M.kv_append_dev(gpu, c.cache, b, None, None, c.ldq, 4, None, c.ldq, None, c.ldk, None, c.ldk)


# ------------------------------------------------- streams, graphs, workspaces
@pytest.mark.parametrize("new", [[1] * 6, [120, 60]])
def test_two_streams_with_a_workspace_each(gpu, new):
    import torch
    cs = [Case("f16", 128, 16, 2, 16, new, [n + 5000 for n in new], seed=s) for s in range(2)]
    refs = [c.attend(gpu) for c in cs]
    streams = [torch.cuda.Stream() for _ in cs]
    need = M.kv_attention_ws_bytes(gpu, cs[0].cache, cs[0].batch, 16)
    wss = [torch.empty(max(need, 16), dtype=torch.uint8, device="cuda") for _ in cs]
    outs = [torch.empty_like(r) for r in refs]
    torch.cuda.synchronize()
    for _ in range(20):
        for c, st, ws, out in zip(cs, streams, wss, outs):
            M.kv_attention_dev(gpu, c.cache, c.batch, c.q.data_ptr(), c.ldq, 16, out.data_ptr(), c.ldq, 128 ** -0.5,
                               ws=ws.data_ptr(), ws_bytes=need, stream=st.cuda_stream)
    torch.cuda.synchronize()
    for c, out, ref in zip(cs, outs, refs):
        assert torch.equal(out[:c.real], ref[:c.real])


def test_graph_of_append_and_attention(gpu):
    """One captured step of a serving loop, replayed as the sequences grow (the tables change in place), eager calls of
    the same thread in between; then a larger eager call that grows the thread's workspace, and the graph again."""
    import torch
    prep = preps(64)["both"]
    dev = {n: torch.from_numpy(np.asarray(prep[n])).cuda() for n in ("qn", "kn", "freq")}
    p = M.kv_prep(dev["qn"].data_ptr(), dev["kn"].data_ptr(), prep["eps"], 64, False, dev["freq"].data_ptr())
    c = Case("f16", 64, 8, 2, 16, [1] * 3, [700, 290, 40], max_len=700)
    old = [690, 280, 30]
    c.length = list(old)
    c.upload()
    out, q2 = torch.empty_like(c.q), torch.empty_like(c.q)
    stream = torch.cuda.Stream()

    def step(st):
        M.kv_append_dev(gpu, c.cache, c.batch, p, c.q.data_ptr(), c.ldq, 8, q2.data_ptr(), c.ldq, c.k.data_ptr(), c.ldk,
                        c.v.data_ptr(), c.ldk, st)
        M.kv_attention_dev(gpu, c.cache, c.batch, q2.data_ptr(), c.ldq, 8, out.data_ptr(), c.ldq, 0.125, stream=st)

    torch.cuda.synchronize()
    step(stream.cuda_stream)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        step(stream.cuda_stream)
    pool = c.k_pool.clone(), c.v_pool.clone()
    for i in range(1, 9):
        if i == 5:
            big = Case("f16", 64, 64, 2, 16, [1] * 40, [4000] * 40)
            big.attend(gpu)
        c.q.normal_()
        c.k.normal_()
        c.v.normal_()
        c.d_len.copy_(torch.tensor([n + i for n in old], dtype=torch.int32))
        c.k_pool.copy_(pool[0])
        c.v_pool.copy_(pool[1])
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got, k, v = out.clone(), c.k_pool.clone(), c.v_pool.clone()
        c.k_pool.copy_(pool[0])
        c.v_pool.copy_(pool[1])
        out.zero_()
        torch.cuda.synchronize()
        step(stream.cuda_stream)
        torch.cuda.synchronize()
        assert torch.equal(got, out) and torch.equal(k, c.k_pool) and torch.equal(v, c.v_pool), i
        pool = k, v


def test_threads_have_their_own_workspace(gpu):
    import torch
    cs = [Case("bf16", 64, 8, 2, 16, [1] * 4, [3000, 20, 800, 1200], seed=s) for s in range(3)]
    refs = [c.attend(gpu) for c in cs]
    bad = []

    def work(c, ref):
        out = torch.empty_like(ref)
        for _ in range(20):
            M.kv_attention_dev(gpu, c.cache, c.batch, c.q.data_ptr(), c.ldq, 8, out.data_ptr(), c.ldq, 0.125)
        torch.cuda.synchronize()
        if not torch.equal(out[:c.real], ref[:c.real]):
            bad.append(c)

    ts = [threading.Thread(target=work, args=a) for a in zip(cs, refs)]
    for t in ts:
        t.start()
    for t in ts:
        t.join()
    assert not bad


# -------------------------------------------------------- as they are used
@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("window,sinks", [(0, 0), (24, 2)])
def test_prompts_then_tokens(gpu, typ, window, sinks):
    """Two sequences' prompts in parts, then token by token: q/k/v products of resident weights, append, attention, output
    product, against the whole computed in 64 bits from the dequantized weights. The cache's rounding is the oracle's too
    (k and v are taken from it), so the bar is that of the products, 1e-4 |ref| + 1e-6 per product, times a few."""
    import torch
    d, heads, kv, dk, page = 256, 4, 2, 64, 16
    r = np.random.default_rng(9)
    names = {"q": heads * dk, "k": kv * dk, "v": kv * dk}
    ws = {n: M.Weight.make(gpu, M.Q8_0, (r.standard_normal((m, d)) * 0.06).astype(np.float32)) for n, m in names.items()}
    ws["o"] = M.Weight.make(gpu, M.Q8_0, (r.standard_normal((d, heads * dk)) * 0.06).astype(np.float32))
    dense = {n: M.host_dequant(gpu, w).astype(np.float64) for n, w in ws.items()}
    dev = {n: M.DeviceWeight(gpu, w) for n, w in ws.items()}
    prep = preps(dk)["both"]
    pd = {n: torch.from_numpy(np.asarray(prep[n])).cuda() for n in ("qn", "kn", "freq")}
    p = M.kv_prep(pd["qn"].data_ptr(), pd["kn"].data_ptr(), prep["eps"], dk, False, pd["freq"].data_ptr())
    total = [75, 40]
    x = [r.standard_normal((n, d)).astype(np.float32) for n in total]
    c = Case(typ, dk, heads, kv, page, [0, 0], total)
    done, outs = [0, 0], [[], []]
    for part in [(50, 20), (17, 10), (3, 0)] + [(1, 1)] * 5 + [(0, 5)]:
        rows = sum(part)
        c.starts, c.length = [0, part[0], rows], [a + b for a, b in zip(done, part)]
        c.rows, c.max_new, c.max_len = rows, max(part), max(c.length)
        c.upload()
        xs = torch.from_numpy(np.concatenate([x[b][done[b]:done[b] + part[b]] for b in (0, 1)])).cuda()
        q, k, v = (torch.empty(rows, m, device="cuda") for m in names.values())
        o, y = torch.empty_like(q), torch.empty(rows, d, device="cuda")
        torch.cuda.synchronize()
        M.qkv_dev(gpu, [dev["q"], dev["k"], dev["v"]], xs.data_ptr(), [q.data_ptr(), k.data_ptr(), v.data_ptr()], rows)
        M.kv_append_dev(gpu, c.cache, c.batch, p, q.data_ptr(), heads * dk, heads, q.data_ptr(), heads * dk, k.data_ptr(),
                        kv * dk, v.data_ptr(), kv * dk)
        M.kv_attention_dev(gpu, c.cache, c.batch, q.data_ptr(), heads * dk, heads, o.data_ptr(), heads * dk, dk ** -0.5, 1,
                           window, sinks)
        dev["o"].gemm(o.data_ptr(), y.data_ptr(), rows)
        torch.cuda.synchronize()
        y = f64(y)
        for b in (0, 1):
            outs[b].append(y[c.starts[b]:c.starts[b + 1]])
            done[b] += part[b]
    assert done == total
    for b, n in enumerate(total):
        x64 = x[b].astype(np.float64)
        q = (x64 @ dense["q"].T).reshape(n, heads, dk)
        q = np.stack([[O.prepare_head(q[t, h], prep["qn"], prep["eps"], t, dk, False, prep["freq"]) for h in range(heads)]
                      for t in range(n)])
        k = (x64 @ dense["k"].T).reshape(n, kv, dk)
        k = np.stack([[O.prepare_head(k[t, h], prep["kn"], prep["eps"], t, dk, False, prep["freq"]) for h in range(kv)]
                      for t in range(n)])
        pg, sl = [int(c.pages[b, j // page]) for j in range(n)], [j % page for j in range(n)]
        got_k, got_v = f64(c.k_pool)[pg, :, sl], f64(c.v_pool)[pg, :, sl]
        half = {"f32": 0.0, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}[typ]
        assert (np.abs(got_k - k) <= (half + 1e-4) * np.abs(k) + 2e-5).all()
        assert (np.abs(got_v - (x64 @ dense["v"].T).reshape(n, kv, dk)) <= (half + 1e-4) * np.abs(got_v) + 2e-5).all()
        ref = np.empty((n, heads, dk))
        for t in range(n):
            keys = O.sees(t, t + 1, 1 << 30, True, window, sinks)
            for h in range(heads):
                s = got_k[keys, h // 2] @ q[t, h] * dk ** -0.5
                w = np.exp(s - s.max())
                ref[t, h] = (w / w.sum()) @ got_v[keys, h // 2]
        ref = ref.reshape(n, -1) @ dense["o"].T
        y = np.concatenate(outs[b])
        assert (np.abs(y - ref) <= 4e-4 * np.abs(ref) + 2e-5).all()
        assert np.linalg.norm(y - ref) <= 5e-6 * np.linalg.norm(ref)
    for w in dev.values():
        w.close()


# ------------------------------------ long sums: prompts' keys in one workgroup
# Forty sequences of 33 rows, eight heads: 320 workgroups, more than the chip has CUs, so no tile's keys are split and one
# workgroup's sums reach over all of them.
LONG = [("f32", 128), ("f16", 128), ("bf16", 128), ("f32", 64), ("f16", 64), ("bf16", 64)]


def long_case(typ, dk, n, kind, nseq=40, new=33):
    """All sequences on the same n keys. kind: random; plateau (the first 64 keys' scores 0, all others one score, 0.7 to 5
    powers of two above them); alike (a plateau whose values are all the same, as frames of silence are)."""
    import torch
    c = Case(typ, dk, 8, 8, 64, [new] * nseq, [n] + [1] * (nseq - 1), seed=n, pad=1)
    c.length, c.pages, c.max_len = [n] * nseq, c.pages[:1].expand(nseq, -1).contiguous(), n
    if kind != "random":
        first = c.pages[0, 0].item()
        c.k_pool[:] = 0.5
        c.k_pool[first] = 0.0
        level = torch.linspace(1.0, 7.0, c.rows, device="cuda")[:, None] / dk ** 0.5     # q . k / sqrt(dk) = 0.5 to 3.5
        c.q.mul_(0.01).add_(level)
        if kind == "alike":
            c.v_pool[:] = c.v_pool[:1, :, :1].clone()
    c.upload()
    return c


def definition(c, window=0, sinks=0):
    """[rows, heads, dim] in 64 bits: every sequence's rows over the keys of the first one's pages."""
    import torch
    n, dk, G = c.length[0], c.dk, c.heads // c.kv_heads
    flat = lambda p: p[c.d_pages[0].long()].permute(1, 0, 2, 3).reshape(c.kv_heads, -1, dk)[:, :n].double()   # noqa: E731
    k, v = flat(c.k_pool), flat(c.v_pool)
    r = torch.arange(c.real, device="cuda")
    start = torch.tensor(c.starts, device="cuda")
    seq = torch.bucketize(r, start[1:], right=True)
    p = (n - (start[seq + 1] - start[seq]) + r - start[seq])[:, None]
    j = torch.arange(n, device="cuda")[None]
    hidden = (j > p) | ((j <= p - window) & (j >= sinks)) if window else j > p
    out = torch.empty(c.real, c.heads, dk, dtype=torch.float64, device="cuda")
    for h in range(c.heads):
        s = c.heads_of(c.q, c.heads)[:c.real, h].double() @ k[h // G].T.contiguous() * dk ** -0.5
        out[:, h] = torch.softmax(s.masked_fill_(hidden, -np.inf), 1) @ v[h // G]
    return out


@pytest.mark.parametrize("n", [8200, 32700])
@pytest.mark.parametrize("kind", ["random", "plateau", "alike"])
@pytest.mark.parametrize("typ,dk", LONG)
def test_long_sums(gpu, typ, dk, kind, n):
    """The sums of probabilities and of values over thousands of keys. Independent roundings: the norm's bar, as above.
    Values all alike: the output is that value whatever the scores are, and roundings of a sum may all go one way, so each
    of the sum's steps counts. A part of 64 tiles (f16; else 32) takes 8 (12) a tile into the context, two into the sum of
    probabilities and 4 that sum a tile's; the parts, 1024 keys at least, n / 1024 each; 16 are for the exponential, the
    terms, the reciprocal and its product."""
    say("long sums", typ, dk, kind, n)
    c = long_case(typ, dk, n, kind)
    out = c.attend(gpu)
    assert (out[c.real:] == 7.25).all()
    y, ref = c.heads_of(out, 8)[:c.real].double(), definition(c)
    rel = ((y - ref).norm() / ref.norm()).item()
    worst = ((y - ref).abs() / ref.abs()).max().item() / U
    say(f"  norm {rel:.3g}, worst {worst:.4g} u")
    if kind == "alike":
        assert worst <= (64 * 10 if typ == "f16" else 32 * 14) + 20 + n / 512
    else:
        assert rel <= 2.0 ** -19


@pytest.mark.parametrize("n", [1024, 1057, 2047, 2048, 2049, 4096, 4129, 8192, 8225, 9000])
@pytest.mark.parametrize("typ,dk", LONG)
def test_long_sums_in_parts(gpu, typ, dk, n):
    """Lengths around the ends of parts, with and without a window; out in place of q."""
    import torch
    for window, sinks in ((0, 0), (n - 700, 70)):
        say("parts", typ, dk, n, window)
        c = long_case(typ, dk, n, "random")
        out = c.attend(gpu, window=window, sinks=sinks)
        assert (out[c.real:] == 7.25).all()
        y, ref = c.heads_of(out, 8)[:c.real].double(), definition(c, window, sinks)
        assert ((y - ref).norm() / ref.norm()).item() <= 2.0 ** -19
        c.attend(gpu, window=window, sinks=sinks, out=c.q)
        assert torch.equal(c.q[:c.real], out[:c.real])


@pytest.mark.parametrize("typ,dk", LONG)
def test_long_sums_of_split_keys(gpu, typ, dk):
    """A prompt's part on a long cache in eight chunks (64 workgroups a chunk), each longer than a part of its sums."""
    say("split", typ, dk)
    c = Case(typ, dk, 8, 8, 64, [1000], [30000])
    y, ref = c.heads_of(c.attend(gpu), 8).double(), definition(c)
    assert M.kv_attention_ws_bytes(gpu, c.cache, c.batch, 8) == 512 * 128 * 4 * (dk + 2)
    assert ((y - ref).norm() / ref.norm()).item() <= 2.0 ** -19


@pytest.mark.parametrize("typ,dk", LONG)
def test_long_sums_keep_a_nan_where_it_is(gpu, typ, dk):
    """A value that is not finite, in the first part of the sums, the second, or the last rows' own: its feature alone, of the
    rows that see it."""
    import torch
    n = 9000
    c = long_case(typ, dk, n, "random")
    base = c.attend(gpu).view(c.rows, 8, dk)
    for j in (100, 5000, n - 10):
        for bad in SPECIAL:
            say("nan", typ, dk, j, bad)
            at = int(c.pages[0, j // 64]), 3, j % 64, 5
            keep = c.v_pool[at].clone()
            c.v_pool[at] = bad
            out = c.attend(gpu).view(c.rows, 8, dk)
            c.v_pool[at] = keep
            sees = torch.zeros(c.rows, dtype=torch.bool, device="cuda")
            sees[:c.real] = torch.arange(c.real, device="cuda") % 33 + n - 33 >= j
            assert not out[sees, 3, 5].isfinite().any()
            out[sees, 3, 5] = base[sees, 3, 5]
            assert torch.equal(out, base)


# --------------------------------------------- the range that the bound is for
def bound_of(c, scale):
    """What the header allows each row and head, with its floors under the elements of q and k (in float64)."""
    q, k = np.abs(f64(c.heads_of(c.q, c.heads))), np.abs(f64(c.k_pool))
    if c.typ == "f16":
        q = np.maximum(q, 2.0 ** -20 * q.max(-1, keepdims=True))
    else:
        q, k = np.maximum(q, 2.0 ** -100 / abs(scale)), np.maximum(k, 2.0 ** -100)
    _, terms, count, vmax = (x[:c.real] for x in O.attention(k, f64(c.v_pool), c.starts, c.length, c.pages.numpy(), q, scale))
    return U * vmax * (2 * (c.dk + 8) * terms + count / 8 + 400)


RANGES = {"wide rows": ["f16"], "small q": ["bf16", "f32"], "large q": ["bf16", "f32"], "small scale": ["f16", "bf16", "f32"],
          "large scale": ["f16", "bf16", "f32"], "largest q": ["f16", "bf16", "f32"], "smallest v": ["bf16", "f32"]}


@pytest.mark.parametrize("new", [1, 12, 70])
@pytest.mark.parametrize("kind,typ", [(k, t) for k, ts in RANGES.items() for t in ts])
def test_range_of_the_bound(gpu, typ, kind, new):
    """Scores of order 1 from elements at the ends of what the header's bound is stated for."""
    say("range", kind, typ, new)
    c = Case(typ, 64, 4, 2, 16, [new], [new + 90])
    scale = 0.125
    if kind == "wide rows":        # one feature 2^24 times the others; the keys have nothing there
        c.q.mul_(8)
        c.q[:, ::64] *= 2.0 ** 24
        c.k_pool[..., 0] = 0
    elif kind == "small q":        # |scale q| of 2^-95
        c.q.mul_(2.0 ** -92)
        c.k_pool.mul_(2.0 ** 95)
    elif kind == "large q":
        c.q.mul_(2.0 ** 95)
        c.k_pool.mul_(2.0 ** -92)
    elif kind == "small scale":    # the sizes of q that make up for it
        scale = 2.0 ** -100
        c.q.mul_(2.0 ** 97)
    elif kind == "large scale":
        scale = 2.0 ** 100
        c.q.mul_(2.0 ** -103)
    elif kind == "largest q":      # on keys that have nothing: the values' mean
        c.q.clamp_(-4, 4).mul_(2.0 ** 100)
        c.k_pool.zero_()
    else:
        c.v_pool.mul_(2.0 ** -100)
    y = f64(c.heads_of(c.attend(gpu, scale), 4))[:c.real]
    ref = O.attention(f64(c.k_pool), f64(c.v_pool), c.starts, c.length, c.pages.numpy(), f64(c.heads_of(c.q, 4)), scale)[0]
    err = np.abs(y - ref[:c.real]).max(-1)
    lim = bound_of(c, scale)
    say(f"  worst {(err / lim).max():.3g} of the bound")
    assert np.isfinite(y).all() and (err <= lim).all()


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("new", [1, 12, 70])
def test_infinite_scores(gpu, typ, new):
    """Keys of -infinity under positive queries: of a row that sees others too, they take nothing or make it NaN; a row
    that sees nothing else is 0 or NaN, never a value. Of +infinity: NaN."""
    import torch
    say("infinite scores", typ, new)
    c = Case(typ, 64, 4, 2, 16, [new], [new + 40])
    c.q.abs_().add_(0.01)
    c.v_pool.abs_().add_(1.0)
    c.k_pool[:] = -float("inf")
    y = c.attend(gpu)
    assert ((y == 0) | y.isnan()).all()
    first = c.pages[0, 0].item()
    c.k_pool[first] = 0.5
    base = c.attend(gpu, causal=0)
    held = c.length
    c.length, c.starts = [16], [0, min(new, 16)]         # the same rows on the finite keys alone
    c.upload()
    few = c.attend(gpu, causal=0)[:min(new, 16)]
    c.length, c.starts = held, [0, new]
    c.upload()
    got = base[:min(new, 16)]
    size = 0.125 * 0.5 * c.heads_of(c.q, 4).sum(-1).max().item()      # the header's A; each of the two is within its bound
    lim = 2 * U * c.v_pool.max().item() * (2 * 72 * size + 16 / 8 + 400)
    assert (got.isnan() | ((got - few).abs() <= lim)).all()
    c.k_pool[first, :, 3] = float("inf")
    assert c.attend(gpu, causal=0).isnan().all()


# ---------------------------------------------------------- the append's edges
@pytest.mark.parametrize("power", [-145, -140, -126, -60, 125])
def test_append_norm_of_all_sizes(gpu, power):
    """Heads of subnormal elements and of ones near f32's largest, without eps: the norm brings both to 1."""
    say("norm", power)
    c = Case("f32", 64, 4, 2, 16, [3, 5], [30, 5])
    c.q.mul_(2.0 ** (power // 2)).mul_(2.0 ** (power - power // 2))
    c.k.mul_(2.0 ** (power // 2)).mul_(2.0 ** (power - power // 2))
    run_append(gpu, c, dict(preps(64)["both"], eps=0.0))


def test_append_norm_of_what_is_not_finite(gpu):
    """An infinity or a NaN makes its head NaN, and no other; so does a head of zeros without eps."""
    import torch
    prep = preps(64)["norm"]
    qn, kn = (torch.from_numpy(prep[n]).cuda() for n in ("qn", "kn"))
    p = M.kv_prep(qn.data_ptr(), kn.data_ptr(), 0.0)
    c = Case("f32", 64, 4, 2, 16, [3], [3])
    outs = []
    for bad in [None] + SPECIAL + [0.0]:
        q = c.q.clone()
        if bad is not None:
            q[1, 64 if bad == 0.0 else 70:128 if bad == 0.0 else 71] = bad
        out = torch.full_like(q, 7.25)
        torch.cuda.synchronize()
        M.kv_append_dev(gpu, c.cache, c.batch, p, q.data_ptr(), c.ldq, 4, out.data_ptr(), c.ldq, c.k.data_ptr(), c.ldk,
                        c.v.data_ptr(), c.ldk)
        torch.cuda.synchronize()
        if bad is not None:
            assert out[1, 64:128].isnan().all()
            out[1, 64:128] = outs[0][1, 64:128]
        outs.append(out)
        assert torch.equal(out, outs[0]) and out.isfinite().all()


@pytest.mark.parametrize("typ,dk", LONG)
@pytest.mark.parametrize("prep", ["norm", "both", "part", "inter"])
def test_append_without_q_prepares_k(gpu, typ, dk, prep):
    """n_heads 0 with a norm and a rotation of k: the bits that the whole call writes, which are right."""
    import torch
    say("append without q", typ, dk, prep)
    c = Case(typ, dk, 6, 2, 7, [3, 0, 1, 12], [10, 5, 1, 12], pad=3, ldx=8)
    pools = c.k_pool.clone(), c.v_pool.clone()
    run_append(gpu, c, preps(dk)[prep])
    whole = c.k_pool.clone(), c.v_pool.clone()
    c.k_pool.copy_(pools[0])
    c.v_pool.copy_(pools[1])
    spec = preps(dk)[prep]
    dev = {n: torch.from_numpy(np.asarray(spec[n])).cuda() for n in ("qn", "kn", "freq") if spec.get(n) is not None}
    ptr = {n: dev[n].data_ptr() if n in dev else None for n in ("qn", "kn", "freq")}
    p = M.kv_prep(ptr["qn"], ptr["kn"], spec.get("eps", 0.0), spec.get("rot", 0), spec.get("interleaved", False), ptr["freq"])
    torch.cuda.synchronize()
    M.kv_append_dev(gpu, c.cache, c.batch, p, None, 0, 0, None, 0, c.k.data_ptr(), c.ldk, c.v.data_ptr(), c.ldk)
    torch.cuda.synchronize()
    assert torch.equal(c.k_pool, whole[0]) and torch.equal(c.v_pool, whole[1])


# ------------------------------------------------------------- mixed batches
@pytest.mark.parametrize("typ,dk", LONG)
@pytest.mark.parametrize("window,sinks", [(0, 0), (600, 5)])
def test_prompts_and_tokens_in_one_call(gpu, typ, dk, window, sinks):
    """A prompt, single tokens on long and short caches and a few rows: one form for all, its keys split over chunks that
    the shorter sequences do not have."""
    say("mixed", typ, dk, window)
    c = Case(typ, dk, 8, 2, 16, [130, 1, 1, 0, 3], [130, 3000, 40, 7, 900], pad=2)
    assert M.kv_attention_ws_bytes(gpu, c.cache, c.batch, 8, 1, window, sinks) > 0
    c.check(gpu, window=window, sinks=sinks)


@pytest.mark.parametrize("typ,dk", LONG)
def test_windowed_parts_of_several_sequences(gpu, typ, dk):
    say("windowed parts", typ, dk)
    c = Case(typ, dk, 2, 1, 25, [300, 200, 90], [2300, 1800, 90], pad=2)
    assert M.kv_attention_ws_bytes(gpu, c.cache, c.batch, 2, 1, 700, 5) > 0
    c.check(gpu, window=700, sinks=5)
