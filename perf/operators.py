"""The paged key-value cache operators, as cases that can be timed.

  append     head norms of q and k, the position rotation, and the
             append of k and v to a paged cache                     mynah_asr_hip_kv_append_dev
  attention  new rows against the cache: one token a sequence, a
             few, or whole prompts; grouped heads, causal or not,
             sliding window with first tokens that stay visible     mynah_asr_hip_kv_attention_dev

Activations are f32, as everywhere in this framework; the cache holds f32, f16
or bf16. `run` computes the operators in elementary torch operations, or, with
`own`, by the framework's calls; `exact` is their definition in 64 bits.

A case's sequences have `new` rows each (new_lo to new_hi, spread over the
logarithm) on top of `old` cached ones; the lengths follow from the case alone,
the values, the rotation's page order and all else from the seed.
"""
import math
import os
import random
import sys

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-6
ROT_BASE = 10000.0


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # --- append
        # one token for each of four requests, model width 1024: the smallest call, launches and latency
        {"name": "append_step_4", "op": "append", "type": "f32", "nseq": 4, "new_lo": 1, "new_hi": 1, "old_lo": 20,
         "old_hi": 400, "heads": 8, "kv_heads": 8, "dim": 128, "page": 16, "norm": True, "rot": 128, "inter": False,
         "packed": False, "pad": 0},
        # one token for each of 256 requests, grouped heads
        {"name": "append_step_256", "op": "append", "type": "bf16", "nseq": 256, "new_lo": 1, "new_hi": 1, "old_lo": 100,
         "old_hi": 60000, "heads": 32, "kv_heads": 8, "dim": 128, "page": 16, "norm": True, "rot": 128, "inter": False,
         "packed": True, "pad": 0},
        # a batch of ragged prompts from a packed q/k/v buffer with rows behind the last sequence; half of each head
        # rotated, in neighbouring pairs
        {"name": "append_prompts", "op": "append", "type": "f16", "nseq": 12, "new_lo": 150, "new_hi": 2500, "old_lo": 0,
         "old_hi": 0, "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "norm": True, "rot": 64, "inter": True,
         "packed": True, "pad": 77},
        # --- attention, single tokens
        # one request's token over a short context: latency
        {"name": "step_1x200", "op": "attention", "type": "f16", "nseq": 1, "new_lo": 1, "new_hi": 1, "old_lo": 199,
         "old_hi": 199, "heads": 8, "kv_heads": 8, "dim": 128, "page": 16, "causal": True, "window": 0, "sinks": 0,
         "pad": 0},
        # a batch of ordinary requests, ragged lengths
        {"name": "step_48_ragged", "op": "attention", "type": "f16", "nseq": 48, "new_lo": 1, "new_hi": 1, "old_lo": 500,
         "old_hi": 9000, "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "causal": True, "window": 0, "sinks": 0,
         "pad": 0},
        # one request over a very long context: split over its length and joined
        {"name": "step_1x131k", "op": "attention", "type": "bf16", "nseq": 1, "new_lo": 1, "new_hi": 1, "old_lo": 131006,
         "old_hi": 131006, "heads": 64, "kv_heads": 8, "dim": 128, "page": 32, "causal": True, "window": 0, "sinks": 0,
         "pad": 0},
        # long requests of a model with a sliding window and four first tokens that stay
        {"name": "step_64_window", "op": "attention", "type": "bf16", "nseq": 64, "new_lo": 1, "new_hi": 1,
         "old_lo": 1000, "old_hi": 30000, "heads": 32, "kv_heads": 8, "dim": 128, "page": 16, "causal": True,
         "window": 4096, "sinks": 4, "pad": 0},
        # four hypotheses of each of 16 utterances over its 750 encoder frames (60 s): cross-attention, f32 cache
        {"name": "cross_16x750", "op": "attention", "type": "f32", "nseq": 16, "new_lo": 4, "new_hi": 4, "old_lo": 746,
         "old_hi": 746, "heads": 8, "kv_heads": 8, "dim": 128, "page": 25, "causal": False, "window": 0, "sinks": 0,
         "pad": 0},
        # --- attention, prompts
        # one long prompt: the largest
        {"name": "prompt_8192", "op": "attention", "type": "f16", "nseq": 1, "new_lo": 8192, "new_hi": 8192, "old_lo": 0,
         "old_hi": 0, "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "causal": True, "window": 0, "sinks": 0,
         "pad": 0},
        # a batch of ragged prompts, heads of 64, rows behind the last sequence
        {"name": "prompts_ragged", "op": "attention", "type": "bf16", "nseq": 8, "new_lo": 100, "new_hi": 4000,
         "old_lo": 0, "old_hi": 0, "heads": 16, "kv_heads": 4, "dim": 64, "page": 16, "causal": True, "window": 0,
         "sinks": 0, "pad": 50},
        # the next part of a prompt that is taken in parts
        {"name": "part_512_on_24k", "op": "attention", "type": "f16", "nseq": 1, "new_lo": 512, "new_hi": 512,
         "old_lo": 24001, "old_hi": 24001, "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "causal": True,
         "window": 0, "sinks": 0, "pad": 0},
        # prompts of a model with a sliding window and first tokens that stay, width 1024, f32 cache
        {"name": "prompts_window", "op": "attention", "type": "f32", "nseq": 4, "new_lo": 700, "new_hi": 3500,
         "old_lo": 0, "old_hi": 500, "heads": 8, "kv_heads": 8, "dim": 128, "page": 16, "causal": True, "window": 512,
         "sinks": 4, "pad": 0},
    ]


def _between(rng, lo, hi):
    """A size spread over the logarithm of [lo, hi]."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    heads, kv_heads = rng.choice([(8, 8), (16, 4), (32, 8), (28, 4), (64, 8), (10, 2), (16, 1)])
    c = {"op": rng.choice(["append", "append", "attention", "attention", "attention", "attention"]),
         "type": rng.choice(["f32", "f16", "bf16", "f16", "bf16"]), "heads": heads, "kv_heads": kv_heads,
         "dim": rng.choice([128, 128, 64]), "page": rng.choice([16, 16, 32, 64, 25, 256])}
    if c["op"] == "append":
        step = rng.random() < 0.5
        c["nseq"] = _between(rng, 1, 512) if step else _between(rng, 1, 16)
        c["new_lo"], c["new_hi"] = (1, 1) if step else sorted(_between(rng, 2, 8192 // c["nseq"]) for _ in range(2))
        c["old_lo"], c["old_hi"] = sorted(_between(rng, 1, 100000 if step else 2000) for _ in range(2))
        c["norm"], c["inter"], c["packed"] = rng.random() < 0.6, rng.random() < 0.5, rng.random() < 0.5
        c["rot"] = rng.choice([c["dim"], c["dim"], c["dim"] // 2, 0])
        c["pad"] = rng.choice([0, 0, 5])
        return c
    form = rng.choice(["step", "step", "few", "prompt", "prompt"])
    if form == "prompt":
        c["nseq"] = _between(rng, 1, 8)
        c["new_lo"], c["new_hi"] = sorted(_between(rng, 17, 6000 // c["nseq"]) for _ in range(2))
        c["old_lo"], c["old_hi"] = sorted(_between(rng, 1, 2000) for _ in range(2))
        c["heads"], c["kv_heads"] = min(heads, 32), kv_heads if heads <= 32 else 4
    else:
        c["nseq"] = _between(rng, 1, 64)
        c["new_lo"], c["new_hi"] = (1, 1) if form == "step" else (1, rng.choice([2, 4, 8]))
        c["old_lo"], c["old_hi"] = sorted(_between(rng, 1, min(100000, 300000 // c["nseq"])) for _ in range(2))
    windowed = rng.random() < 0.35
    c["causal"] = windowed or rng.random() < 0.8
    c["window"] = _between(rng, 16, 4096) if windowed else 0
    c["sinks"] = rng.choice([0, 1, 4, 64]) if windowed else 0
    c["pad"] = rng.choice([0, 0, 3])
    return c


def _lengths(case):
    """(new rows, cached rows before them) of each sequence."""
    r = random.Random("%(nseq)d %(new_lo)d %(new_hi)d %(old_lo)d %(old_hi)d" % case)

    def spread(lo, hi):
        return lo if lo == hi else max(lo, min(hi, int(math.exp(r.uniform(math.log(max(lo, 1)), math.log(hi))))))

    return [(spread(case["new_lo"], case["new_hi"]), spread(case["old_lo"], case["old_hi"])) for _ in range(case["nseq"])]


# ----------------------------------------------------------------- the inputs
def prepare(case, seed):
    """What a serving loop holds before the call: the cache, the batch's tables and the rows of q, k and v. With `own` on the
    default stream, the current stream becomes one that the framework can be given, as a program sets it up once: inputs,
    calls and what reads their outputs are then in order without waits."""
    if own and not torch.cuda.current_stream().cuda_stream:
        _framework()
        torch.cuda.set_stream(_stream)
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt, hq, hk, dk, page = TYPES[case["type"]], case["heads"], case["kv_heads"], case["dim"], case["page"]
    lengths = _lengths(case)
    total = [n + o for n, o in lengths]
    starts = [0]
    for n, _ in lengths:
        starts.append(starts[-1] + n)
    real = starts[-1]
    rows = real + case["pad"]

    def normal(*shape, sigma=1.0, dtype=torch.float32):
        return torch.randn(*shape, generator=g, device="cuda", dtype=dtype).mul_(sigma)

    append = case["op"] == "append"
    # an append touches its rows' pages alone, so its pool holds those: a sequence's pages before them are shared ones
    first = [o // page if append else 0 for _, o in lengths]
    need = [-(-t // page) - f for t, f in zip(total, first)]
    most = max(-(-t // page) for t in total)
    n_pages = sum(need) + 3
    order = torch.randperm(n_pages, generator=g, device="cuda").int().cpu()
    table = torch.full((len(total), most), int(order[-1]), dtype=torch.int32)
    at = 0
    for b, (f, m) in enumerate(zip(first, need)):
        table[b, f:f + m] = order[at:at + m]
        at += m
    s = {"case": case, "dim": dk, "heads": hq, "kv_heads": hk, "page": page, "real": real, "rows": rows,
         "max_new": max(n for n, _ in lengths), "max_len": max(total), "n_pages": n_pages,
         "row_start": torch.tensor(starts, dtype=torch.int32).cuda(), "len": torch.tensor(total, dtype=torch.int32).cuda(),
         "pages": table.cuda(),
         "k_cache": normal(n_pages, hk, page, dk, dtype=dt), "v_cache": normal(n_pages, hk, page, dk, dtype=dt)}
    if append:
        if case["packed"]:   # one buffer of a fused product: [q heads | k heads | v heads | padding]
            x = normal(rows, (hq + 2 * hk) * dk + 8)
            s["q"], s["k"], s["v"], _ = x.split([hq * dk, hk * dk, hk * dk, 8], 1)
        else:
            s["q"], s["k"], s["v"] = normal(rows, hq * dk), normal(rows, hk * dk), normal(rows, hk * dk)
        s["q_out"] = normal(rows, hq * dk)
        s["q_norm"] = normal(dk, sigma=0.2).add_(1) if case["norm"] else None
        s["k_norm"] = normal(dk, sigma=0.2).add_(1) if case["norm"] else None
        rot = case["rot"]
        s["freq"] = ROT_BASE ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot).cuda() if rot else None
    else:
        s["q"], s["out"] = normal(rows, hq * dk, sigma=2.0), normal(rows, hq * dk)
        s["scale"] = dk ** -0.5
    if own:
        s.update(_handles(s))
    torch.cuda.synchronize()
    return s


def run(s):
    if own:
        return _append_own(s) if s["case"]["op"] == "append" else _attention_own(s)
    return _append_plain(s) if s["case"]["op"] == "append" else _attention_plain(s)


# ------------------------------------------------------ the framework's calls
_lib = _stream = None


def _framework():
    global _lib, _stream
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mynah-asr_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    import mynah_hip as M
    if _lib is None:
        _lib, _stream = M.HipLib(), torch.cuda.Stream()
    return M


def _current(device):
    """The handle of the current stream (what torch.cuda.current_stream(device).cuda_stream gives, which takes 3 us)."""
    return torch._C._cuda_getCurrentRawStream(device)


def _on_a_stream(s, call):
    """call(handle) in the order of the caller's current stream. The framework takes 0, the handle of torch's default
    stream, for the thread's own stream; from there the call goes by a stream between two waits."""
    handle = _current(s["device"])
    if handle:
        call(handle)
        return
    here = torch.cuda.current_stream(s["device"])
    _stream.wait_stream(here)
    call(_stream.cuda_stream)
    here.wait_stream(_stream)


def _handles(s):
    """The descriptions of the cache and the batch that a program makes once."""
    M = _framework()
    c = s["case"]
    kind = {"f32": M.F32, "f16": M.F16, "bf16": M.BF16}[c["type"]]
    h = {"M": M, "device": s["q"].device.index,
         "cache": M.kv_cache(kind, s["k_cache"].data_ptr(), s["v_cache"].data_ptr(), s["n_pages"], s["page"], s["kv_heads"],
                             s["dim"]),
         "batch": M.kv_batch(s["row_start"].data_ptr(), s["len"].data_ptr(), s["pages"].data_ptr(), c["nseq"], s["rows"],
                             s["pages"].shape[1], s["max_new"], s["max_len"])}
    if c["op"] == "append":
        ptr = {n: s[n].data_ptr() if s[n] is not None else None for n in ("q_norm", "k_norm", "freq")}
        h["prep"] = M.kv_prep(q_norm=ptr["q_norm"], k_norm=ptr["k_norm"], eps=EPS, rot=c["rot"], interleaved=c["inter"],
                              freq=ptr["freq"])
    return h


def _append_own(s):
    _on_a_stream(s, lambda stream: s["M"].kv_append_dev(
        _lib, s["cache"], s["batch"], s["prep"], s["q"].data_ptr(), s["q"].stride(0), s["heads"], s["q_out"].data_ptr(),
        s["q_out"].stride(0), s["k"].data_ptr(), s["k"].stride(0), s["v"].data_ptr(), s["v"].stride(0), stream))
    return {"q": s["q_out"], "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _attention_own(s):
    c = s["case"]
    _on_a_stream(s, lambda stream: s["M"].kv_attention_dev(
        _lib, s["cache"], s["batch"], s["q"].data_ptr(), s["q"].stride(0), s["heads"], s["out"].data_ptr(),
        s["out"].stride(0), s["scale"], int(c["causal"]), c["window"], c["sinks"], stream=stream))
    return s["out"]


# ------------------------------------------------------------- the plain forms
def _rows_of(s):
    """[real] the sequence of each row and its position."""
    r = torch.arange(s["real"], device="cuda")
    seq = torch.bucketize(r, s["row_start"][1:].long(), right=True)
    start = s["row_start"].long()
    return seq, s["len"].long()[seq] - (start[seq + 1] - start[seq]) + r - start[seq]


def _head_norm(x, w):
    return x if w is None else x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w


def _rotate(x, cos, sin, rot, inter):
    """x [rows, heads, dim], its first `rot` features turned; cos and sin [rows, 1, rot / 2]."""
    y, rest = x[..., :rot], x[..., rot:]
    a, b = (y[..., 0::2], y[..., 1::2]) if inter else (y[..., :rot // 2], y[..., rot // 2:])
    u, v = a * cos - b * sin, a * sin + b * cos
    y = torch.stack((u, v), -1).flatten(-2) if inter else torch.cat((u, v), -1)
    return torch.cat((y, rest), -1)


def _append_plain(s):
    c, n, dk = s["case"], s["real"], s["dim"]
    seq, pos = _rows_of(s)
    q = _head_norm(s["q"][:n].reshape(n, -1, dk), s["q_norm"])
    k = _head_norm(s["k"][:n].reshape(n, -1, dk), s["k_norm"])
    if c["rot"]:
        angle = pos.double()[:, None, None] * s["freq"]   # (64 bits: far positions)
        cos, sin = angle.cos().float(), angle.sin().float()
        q, k = (_rotate(x, cos, sin, c["rot"], c["inter"]) for x in (q, k))
    s["q_out"][:n] = q.reshape(n, -1)
    page, slot = s["pages"][seq, pos // s["page"]].long(), pos % s["page"]
    s["k_cache"][page, :, slot] = k.to(s["k_cache"].dtype)
    s["v_cache"][page, :, slot] = s["v"][:n].reshape(n, -1, dk).to(s["v_cache"].dtype)
    return {"q": s["q_out"], "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _attention_plain(s):
    c, dk, hk = s["case"], s["dim"], s["kv_heads"]
    nseq, G, N, L = c["nseq"], s["heads"] // hk, s["max_new"], s["max_len"]
    start, length = s["row_start"].long(), s["len"].long()
    i = torch.arange(N, device="cuda")[None]
    live = i < (start[1:] - start[:-1])[:, None]                        # [nseq, N] padded rows
    row = torch.where(live, start[:-1, None] + i, 0)
    pos = (length - (start[1:] - start[:-1]))[:, None] + i
    j = torch.arange(L, device="cuda")
    page = s["pages"].long()[:, j // s["page"]]                         # [nseq, L]
    k = s["k_cache"][page, :, j % s["page"]].float().permute(0, 2, 1, 3).reshape(nseq * hk, L, dk)
    v = s["v_cache"][page, :, j % s["page"]].float().permute(0, 2, 1, 3).reshape(nseq * hk, L, dk)
    q = s["q"][row].reshape(nseq, N, hk, G, dk).permute(0, 2, 1, 3, 4).reshape(nseq * hk, N * G, dk)
    see = (j < length[:, None]).expand(nseq, L)[:, None]                # [nseq, N, L]
    if c["causal"]:
        see = see & (j <= pos[..., None])
    if c["window"]:
        see = see & ((j > pos[..., None] - c["window"]) | (j < c["sinks"]))
    see = see.expand(nseq, N, L)[:, None, :, None]
    x = torch.bmm(q, k.transpose(1, 2).contiguous()).mul_(s["scale"]).view(nseq, hk, N, G, L)
    x = x.masked_fill_(~see, -math.inf)
    x = x.sub_(x.amax(-1, keepdim=True).clamp_min(-3e38)).exp_()
    total = x.sum(-1, keepdim=True)
    y = torch.bmm(x.view(nseq * hk, N * G, L), v).view(nseq, hk, N, G, dk) / total.clamp_min(1e-30)
    s["out"][row[live]] = y.permute(0, 2, 1, 3, 4).reshape(nseq, N, -1)[live]
    return s["out"]


# ------------------------------------------------------ their definition in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return _exact_append(s) if case["op"] == "append" else _exact_attention(s)


def _exact_append(s):
    c, dk, page = s["case"], s["dim"], s["page"]
    q_out, kc, vc = s["q_out"].double(), s["k_cache"].double(), s["v_cache"].double()
    starts, lens, pages = s["row_start"].tolist(), s["len"].tolist(), s["pages"].long()
    for b, length in enumerate(lens):
        r0, r1 = starts[b], starts[b + 1]
        p = torch.arange(length - (r1 - r0), length, device="cuda")
        got = []
        for name in ("q", "k"):
            x = s[name][r0:r1].double().view(r1 - r0, -1, dk)
            if c["norm"]:
                x = x / ((x ** 2).sum(-1, keepdim=True) / dk + EPS).sqrt() * s[name + "_norm"].double()
            half = c["rot"] // 2
            if half:   # a pair is a complex number, turned by exp(i angle)
                at = torch.arange(half, device="cuda")
                a, b2 = (2 * at, 2 * at + 1) if c["inter"] else (at, at + half)
                z = torch.complex(x[..., a], x[..., b2]) * torch.exp(1j * p[:, None, None].double() * s["freq"])
                x = x.clone()
                x[..., a], x[..., b2] = z.real, z.imag
            got.append(x)
        q_out[r0:r1] = got[0].reshape(r1 - r0, -1)
        at = pages[b][p // page]
        kc[at, :, p % page] = got[1]
        vc[at, :, p % page] = s["v"][r0:r1].double().view(r1 - r0, -1, dk)
    return {"q": q_out, "k_cache": kc, "v_cache": vc}


def _exact_attention(s):
    c, dk, hk, page = s["case"], s["dim"], s["kv_heads"], s["page"]
    G = s["heads"] // hk
    out = s["out"].double()
    starts, lens = s["row_start"].tolist(), s["len"].tolist()
    for b, length in enumerate(lens):
        r0, r1 = starts[b], starts[b + 1]
        n = r1 - r0
        p = torch.arange(length - n, length, device="cuda")[:, None]
        lo = max(0, length - n - c["window"] + 1) if c["window"] else 0   # the first key in any row's window
        j = torch.arange(lo, length, device="cuda")
        j = torch.cat([torch.arange(min(c["sinks"], lo), device="cuda"), j])
        hidden = torch.zeros(n, len(j), dtype=torch.bool, device="cuda")
        if c["causal"]:
            hidden |= j > p
        if c["window"]:
            hidden |= (j <= p - c["window"]) & (j >= c["sinks"])
        at = s["pages"][b].long()[j // page]
        for h in range(hk):
            k, v = s["k_cache"][at, h, j % page].double(), s["v_cache"][at, h, j % page].double()
            for g in range(G):
                cols = slice((h * G + g) * dk, (h * G + g + 1) * dk)
                w = s["q"][r0:r1, cols].double() @ k.T.contiguous() * s["scale"]
                w = torch.exp(torch.log_softmax(w.masked_fill(hidden, -math.inf), 1))
                out[r0:r1, cols] = w @ v
    return out


# ------------------------------------------------------------------- the work
def work(case):
    size, hq, hk, dk = 4 if case["type"] == "f32" else 2, case["heads"], case["kv_heads"], case["dim"]
    lengths = _lengths(case)
    rows = sum(n for n, _ in lengths)
    if case["op"] == "append":
        return {"bytes": rows * dk * (8 * hq + 2 * hk * (4 + size)),
                "flops": rows * ((hq + hk) * (4 * dk * case["norm"] + 3 * case["rot"]))}
    keys = pairs = 0
    for n, o in lengths:
        p = range(o, o + n)
        w, sinks = case["window"], case["sinks"]
        if w:
            first = max(0, o - w + 1)
            keys += o + n - first + min(sinks, first)
            pairs += sum(min(x + 1, w) + min(sinks, max(0, x + 1 - w)) for x in p)
        else:
            keys += o + n
            pairs += sum(x + 1 for x in p) if case["causal"] else n * (o + n)
    return {"bytes": 2 * keys * hk * dk * size + 8 * rows * hq * dk, "flops": 4 * pairs * hq * dk}
