"""What the rolling cache's operators are timed on: attention over a sliding window with a few
first tokens that stay visible (sinks), and the append that rotates q and k on the way into the
cache.

``run`` makes one call: with ``own`` the framework's (``mini_vllm.kernels.ops``), otherwise the
operator's plain form in elementary torch operations and 32 bits. Shapes are the Qwen3-0.6B ones
of this repository (16 query heads over 8 kv heads, head dim 128, 16-token pages in shuffled
order) and generic wider or narrower ones (32 over 8, one kv head per query head, head dims 64 and
256). K, V and queries are N(0, 1), which is what QK-normed heads hold. The attention cases hold
the pages that a query of the call sees and no others: the table entries of the pages behind the
window are -1, as a server leaves them that gives those pages to other sequences.
"""

import math
import random
import sys
from pathlib import Path

import torch

own = False

DEVICE = "cuda"
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16,
          "fp8": torch.float8_e4m3fn}
BYTES = {"f32": 4, "f16": 2, "bf16": 2, "fp8": 1}
PAGE = 16
THETA = 1_000_000.0
E4M3_MAX = 448.0


# ------------------------------------------------------------------------------- cases


def attend(name, dtype, kv, decodes, lo, hi, chunks, chunk_lo, chunk_hi, prefix_lo, prefix_hi,
           window, sinks, hq=16, hk=8, d=128, layout=0):
    return dict(name=name, kind="attend", dtype=dtype, kv=kv, hq=hq, hk=hk, d=d, decodes=decodes,
                lo=lo, hi=hi, chunks=chunks, chunk_lo=chunk_lo, chunk_hi=chunk_hi,
                prefix_lo=prefix_lo, prefix_hi=prefix_hi, window=window, sinks=sinks,
                layout=layout)


def append(name, dtype, kv, seqs, new_lo, new_hi, prefix_hi, padded=0, hq=16, hk=8, d=128,
           layout=0):
    return dict(name=name, kind="append", dtype=dtype, kv=kv, hq=hq, hk=hk, d=d, seqs=seqs,
                new_lo=new_lo, new_hi=new_hi, prefix_hi=prefix_hi, padded=padded, layout=layout)


def listed():
    return [
        # One user's conversation, long past its window: a decode step for a single sequence,
        # where latency counts.
        attend("decode_bf16_1", "bf16", "bf16", 1, 32000, 32000, 0, 0, 0, 0, 0, 1024, 4),
        # A small float32 model in a test or on a workstation: four short requests, some shorter
        # than the window, head dim 64, a query head per kv head, an odd window.
        attend("decode_f32_4", "f32", "f32", 4, 37, 1000, 0, 0, 0, 0, 0, 333, 1, hq=8, hk=8, d=64),
        # A full decode batch of a server: contexts on both sides of the window.
        attend("decode_bf16_64", "bf16", "bf16", 64, 512, 16384, 0, 0, 0, 0, 0, 1024, 4),
        # The largest decode batch, a wide window over an fp8 cache.
        attend("decode_fp8_256", "bf16", "fp8", 256, 2048, 32768, 0, 0, 0, 0, 0, 4096, 16),
        # Chunked prefill as the scheduler makes it: 512-token chunks after ragged prefixes.
        attend("prefill_bf16_8x512", "bf16", "bf16", 0, 0, 0, 8, 512, 512, 0, 8192, 1024, 4),
        # Whole fresh prompts of a model with windowed layers and no sinks.
        attend("prefill_bf16_fresh", "bf16", "bf16", 0, 0, 0, 4, 4096, 4096, 0, 0, 1024, 0),
        # A long document's last chunk, float16, four query heads per kv head.
        attend("prefill_f16_long", "f16", "f16", 0, 0, 0, 1, 2048, 2048, 30000, 30000, 4096, 4,
               hq=32),
        # An engine iteration over an fp8 cache: ragged chunks beside running decodes.
        attend("mixed_fp8", "bf16", "fp8", 28, 64, 6000, 5, 61, 512, 0, 4000, 700, 5),
        # A decode step's append: one token for each of 32 sequences.
        append("append_bf16_32", "bf16", "bf16", 32, 1, 1, 8192),
        # A prefill iteration's append: ragged chunks, 16-bit pages.
        append("append_bf16_8k", "bf16", "bf16", 8, 700, 1500, 8192, layout=1),
        # A decode step's append over an fp8 cache, a captured batch with padding rows: pages
        # half full, whose scale may grow.
        append("append_fp8_64", "bf16", "fp8", 57, 1, 1, 8192, padded=7, layout=2),
        # A prefill iteration's append over an fp8 cache.
        append("append_fp8_8k", "bf16", "fp8", 8, 700, 1500, 8192, layout=3),
    ]


def draw(rng):
    def near(lo, hi):  # spread over the logarithm
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    hq, hk, d = rng.choice([(16, 8, 128), (16, 8, 128), (16, 8, 128), (32, 8, 128), (8, 8, 128),
                            (12, 4, 128), (16, 4, 64), (8, 2, 256)])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    kv = rng.choice([dtype, "fp8"])
    layout = rng.randrange(1 << 20)
    what = rng.choice(["decode", "decode", "prefill", "prefill", "mixed", "append", "append"])
    if what == "append":
        new = near(1, 1500)
        seqs = min(near(1, 256), max(1, 8192 // new))
        c = append("", rng.choice([dtype, "f32"]), "", seqs, max(1, new // 2), new,
                   near(1, 8192), rng.choice([0, 0, 3]), hq, hk, d, layout)
        c["kv"] = rng.choice([c["dtype"], "fp8"])
    else:
        window, sinks = near(16, 4096), rng.choice([0, 1, 4, 4, 17, 64])
        if what == "decode":
            if rng.random() < 0.25:
                dtype, kv = "f32", rng.choice(["f32", "fp8"])
            n = near(1, 128)
            c = attend("", dtype, kv, n, 1, near(16, 32768), 0, 0, 0, 0, 0, window, sinks, hq, hk,
                       d, layout)
        else:
            longest = near(2, 300 if what == "mixed" else 2048)
            n = min(near(1, 16), max(1, 4096 // longest))
            decodes = near(1, 24) if what == "mixed" else 0
            c = attend("", dtype, kv, decodes, 1, near(64, 8192), n, max(2, longest // 3), longest,
                       0, near(1, 16384), window, sinks, hq, hk, d, layout)
    del c["name"]
    return c


def lengths(c):
    """(context lengths, query lengths) of an attention case's sequences."""
    r = random.Random(c["layout"])
    pairs = [(r.randint(c["lo"], c["hi"]), 1) for _ in range(c["decodes"])]
    for _ in range(c["chunks"]):
        new = r.randint(c["chunk_lo"], c["chunk_hi"])
        pairs.append((r.randint(c["prefix_lo"], c["prefix_hi"]) + new, new))
    r.shuffle(pairs)
    return [s for s, _ in pairs], [n for _, n in pairs]


def additions(c):
    """(prefix, new tokens) of an append case's sequences."""
    r = random.Random(c["layout"])
    return [(r.randint(0, c["prefix_hi"]), r.randint(c["new_lo"], c["new_hi"]))
            for _ in range(c["seqs"])]


# ------------------------------------------------------------------------------- inputs


def randn(shape, g, dtype):
    return torch.randn(shape, generator=g, device=DEVICE).to(dtype)


def fp8_pages(shape, g):
    """An fp8 pool as the framework's write leaves it: codes, and a power-of-two scale for each
    page and kv head."""
    x = torch.randn(shape, generator=g, device=DEVICE)
    scale = torch.exp2(torch.ceil(torch.log2(x.abs().amax(dim=(1, 3)) / E4M3_MAX)))
    return (x / scale[:, None, :, None]).to(torch.float8_e4m3fn), scale


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    return (prepare_attend if case["kind"] == "attend" else prepare_append)(case, seed, g)


def prepare_attend(c, seed, g):
    contexts, new = lengths(c)
    n, window, sinks = len(contexts), c["window"], c["sinks"]
    held = []  # the pages of each sequence that a query of the call sees
    for s, l in zip(contexts, new):
        first = max(0, s - l - window + 1)
        last = -(-s // PAGE)
        front = min(-(-sinks // PAGE), last)
        held.append(list(range(front)) + list(range(max(front, first // PAGE), last)))
    total = sum(map(len, held)) + 3
    order = list(range(total))
    random.Random(seed).shuffle(order)
    tables = torch.full((n, max(-(-s // PAGE) for s in contexts)), -1, dtype=torch.int32)
    at = 0
    for i, pages in enumerate(held):
        tables[i, pages] = torch.tensor(order[at:at + len(pages)], dtype=torch.int32)
        at += len(pages)
    shape = (total, PAGE, c["hk"], c["d"])
    state = {"case": c, "k_scale": None, "v_scale": None}
    if c["kv"] == "fp8":
        state["k"], state["k_scale"] = fp8_pages(shape, g)
        state["v"], state["v_scale"] = fp8_pages(shape, g)
    else:
        state["k"] = randn(shape, g, DTYPES[c["kv"]])
        state["v"] = randn(shape, g, DTYPES[c["kv"]])
    cu = torch.tensor([0, *new]).cumsum(0).to(torch.int32)
    state["q"] = randn((int(cu[-1]), c["hq"], c["d"]), g, DTYPES[c["dtype"]])
    state["tables"] = tables.to(DEVICE)
    state["cu"] = cu.to(DEVICE)
    state["contexts"] = torch.tensor(contexts, dtype=torch.int32).to(DEVICE)
    state["new"] = torch.tensor(new, dtype=torch.int32).to(DEVICE)
    state["longest"], state["furthest"] = max(new), max(contexts)
    return state


def prepare_append(c, seed, g):
    plan = additions(c)
    tokens = sum(l for _, l in plan) + c["padded"]
    first = [p // PAGE for p, _ in plan]
    count = [-(-(p + l) // PAGE) - p // PAGE for p, l in plan]
    total = sum(count) + 3
    order = list(range(total))
    random.Random(seed).shuffle(order)
    slots, positions, at = [], [], 0
    for (p, l), f, k in zip(plan, first, count):
        ids = order[at:at + k]
        at += k
        slots += [ids[j // PAGE - f] * PAGE + j % PAGE for j in range(p, p + l)]
        positions += range(p, p + l)
    slots += [-1] * c["padded"]
    positions += [0] * c["padded"]
    hq, hk, d = c["hq"], c["hk"], c["d"]
    # q, k and v are column views of the one projection that makes them
    fused = randn((tokens, (hq + 2 * hk) * d), g, DTYPES[c["dtype"]])
    q, k, v = fused.split([hq * d, hk * d, hk * d], dim=1)
    far = c["prefix_hi"] + c["new_hi"]
    angles = torch.outer(torch.arange(far, dtype=torch.float64),
                         THETA ** (-torch.arange(0, d, 2, dtype=torch.float64) / d))
    angles = torch.cat((angles, angles), dim=1).to(DEVICE)
    state = {"case": c, "q": q.view(tokens, hq, d), "k": k.view(tokens, hk, d),
             "v": v.view(tokens, hk, d), "k_scale": None, "v_scale": None,
             "positions": torch.tensor(positions, dtype=torch.int64).to(DEVICE),
             "slots": torch.tensor(slots, dtype=torch.int32).to(DEVICE),
             "cos": angles.cos().float(), "sin": angles.sin().float()}
    shape = (total, PAGE, hk, d)
    if c["kv"] == "fp8":
        state["k_pool"], state["k_scale"] = fp8_pages(shape, g)
        state["v_pool"], state["v_scale"] = fp8_pages(shape, g)
    else:
        state["k_pool"] = randn(shape, g, DTYPES[c["kv"]])
        state["v_pool"] = randn(shape, g, DTYPES[c["kv"]])
    return state


# ------------------------------------------------------------------------------- one pass


def run(state):
    if state["case"]["kind"] == "attend":
        return attend_own(state) if own else attend_plain(state)
    if own:
        q = append_own(state)
    else:
        q = append_plain(state)
    return {"q": q, "k": held_values(state["k_pool"], state["k_scale"]),
            "v": held_values(state["v_pool"], state["v_scale"])}


def held_values(pool, scale):
    """What a pool stands for: itself, or codes times their scales (exact in bfloat16, the scales
    being powers of two)."""
    if scale is None:
        return pool
    return pool.to(torch.bfloat16) * scale.to(torch.bfloat16)[:, None, :, None]


PACKAGE = str(Path(__file__).resolve().parent.parent / "mini-vllm_amd")


def the_ops():
    if "mini_vllm" not in sys.modules:
        sys.path.insert(0, PACKAGE)
    from mini_vllm.kernels import ops

    return ops


def attend_own(s):
    c = s["case"]
    return the_ops().paged_window_attention(
        s["q"], s["k"], s["v"], s["tables"], s["cu"], s["contexts"], s["new"], s["longest"],
        s["furthest"], c["window"], c["sinks"], 1.0 / math.sqrt(c["d"]), use_cuda=True,
        k_scale=s["k_scale"], v_scale=s["v_scale"])


def append_own(s):
    return the_ops().rope_kv_write(
        s["q"], s["k"], s["v"], s["positions"], s["cos"], s["sin"], s["k_pool"], s["v_pool"],
        s["slots"], use_cuda=True, k_scale=s["k_scale"], v_scale=s["v_scale"])


def attend_plain(s):
    """Query r of a sequence with S keys and L queries stands at p = S - L + r and sees the keys
    j <= p with j > p - window or j < sinks. All sequences at once, padded to the longest: the key
    axis holds the sinks, then every key from the first query's window on."""
    c = s["case"]
    window, sinks, hq, hk, d = c["window"], c["sinks"], c["hq"], c["hk"], c["d"]
    contexts, new, cu = s["contexts"].long(), s["new"].long(), s["cu"].long()
    n, longest = contexts.numel(), s["longest"]
    base = (contexts - new - window + 1).clamp(min=sinks)[:, None]
    axis = torch.arange(sinks + min(window - 1 + longest, s["furthest"]), device=DEVICE)[None]
    keys = torch.where(axis < sinks, axis, base + axis - sinks)          # n x V positions
    held = keys < contexts[:, None]
    keys = torch.minimum(keys, contexts[:, None] - 1)
    # (a padded or unheld place reads the sequence's last key and is masked)
    pages = s["tables"].long().gather(1, torch.where(held, keys, contexts[:, None] - 1) // PAGE)
    rows = torch.arange(longest, device=DEVICE)[None]
    at = (contexts - new)[:, None] + rows                                # n x L positions
    seen = (held[:, None] & (keys[:, None] <= at[:, :, None])
            & ((keys[:, None] > at[:, :, None] - window) | (keys[:, None] < sinks)))
    k = gathered(s["k"], s["k_scale"], pages, keys % PAGE)               # n x V x hk x d
    v = gathered(s["v"], s["v_scale"], pages, keys % PAGE)
    q_rows = torch.minimum(cu[:-1, None] + rows, cu[1:, None] - 1)
    q = s["q"][q_rows].float().view(n, longest, hk, hq // hk, d)
    q = q.permute(0, 2, 3, 1, 4).reshape(n, hk, -1, d)                   # n x hk x (g L) x d
    scores = q @ k.permute(0, 2, 3, 1).contiguous() * (1.0 / math.sqrt(d))
    scores = scores.view(n, hk, hq // hk, longest, -1)
    scores = scores.masked_fill(~seen[:, None, None], -math.inf)
    weights = torch.exp(scores - scores.amax(dim=-1, keepdim=True))
    weights = weights / weights.sum(dim=-1, keepdim=True)
    out = weights.view(n, hk, -1, weights.shape[-1]) @ v.permute(0, 2, 1, 3).contiguous()
    out = out.view(n, hq, longest, d).permute(0, 2, 1, 3)
    return out[rows < new[:, None]].to(s["q"].dtype)


def gathered(pool, scale, pages, rows):
    x = pool.view(-1, *pool.shape[2:])[pages * PAGE + rows]
    x = x.float()
    return x if scale is None else x * scale[pages][..., None]


def rotated(x, cos, sin):
    """x cos + rotate_half(x) sin at each token's position, in 32 bits."""
    x = x.float()
    low, high = x.chunk(2, dim=-1)
    return x * cos[:, None] + torch.cat((-high, low), dim=-1) * sin[:, None]


def append_plain(s):
    """Rotate q and k; write k and v to their slots (a negative slot writes nothing). An fp8 page
    keeps one power-of-two scale per kv head: the largest that it needed since it was opened by a
    write to its first row, the rows in it re-encoded when it grows."""
    cos, sin = s["cos"][s["positions"]], s["sin"][s["positions"]]
    keep = s["slots"] >= 0
    slots = s["slots"].long()[keep]
    k, v = rotated(s["k"], cos, sin)[keep], s["v"][keep]
    if s["k_scale"] is None:
        s["k_pool"].view(-1, *k.shape[1:])[slots] = k.to(s["k_pool"].dtype)
        s["v_pool"].view(-1, *v.shape[1:])[slots] = v.to(s["v_pool"].dtype)
    else:
        append_fp8(s["k_pool"], s["k_scale"], k, slots)
        append_fp8(s["v_pool"], s["v_scale"], v.float(), slots)
    return rotated(s["q"], cos, sin).to(s["q"].dtype)


def append_fp8(pool, scale, x, slots):
    pages, rows, hk = slots // PAGE, slots % PAGE, pool.shape[2]
    first = torch.full_like(scale[:, 0], PAGE).scatter_reduce(0, pages, rows.float(), "amin")
    most = torch.zeros_like(scale).scatter_reduce(
        0, pages[:, None].expand(-1, hk), x.abs().amax(dim=-1), "amax")
    old = torch.where(first[:, None] > 0, scale, 0.0)
    fraction, exponent = torch.frexp(most / E4M3_MAX)                    # in [0.5, 1) 2^exponent
    need = torch.ldexp((most > 0).float(), exponent - (fraction == 0.5).int())
    new = torch.maximum(old, need)
    before = torch.arange(PAGE, device=DEVICE)[None] < first[:, None]    # rows there already
    ratio = torch.where((old > 0) & (new > old), old / new, 1.0)
    codes = pool.float() * torch.where(before[:, :, None], ratio[:, None], 1.0)[..., None]
    codes.view(-1, *x.shape[1:])[slots] = x / new[pages][..., None]
    pool.copy_(codes.clamp(-E4M3_MAX, E4M3_MAX))
    scale.copy_(new)


# ------------------------------------------------------------------------------- its work


def work(case):
    c = case
    size = BYTES[c["dtype"]]
    if c["kind"] == "append":
        tokens = sum(l for _, l in additions(c))
        row = c["hk"] * c["d"]
        moved = 2 * tokens * c["hq"] * c["d"] * size                     # q in and out
        moved += 2 * tokens * row * (size + BYTES[c["kv"]])              # k and v
        moved += tokens * (8 + 4) + min(tokens, c["prefix_hi"] + c["new_hi"]) * 2 * 4 * c["d"]
        return {"bytes": moved, "flops": 3 * tokens * (c["hq"] + c["hk"]) * c["d"]}
    contexts, new = lengths(c)
    window, sinks = c["window"], c["sinks"]
    keys = pairs = 0
    for s, l in zip(contexts, new):
        first = s - l
        front = min(sinks, s)
        keys += front + max(0, s - max(front, first - window + 1))
        for p in range(first, s):
            pairs += min(p + 1, sinks) + max(0, p + 1 - max(min(p + 1, sinks), p - window + 1))
    moved = 2 * keys * c["hk"] * c["d"] * BYTES[c["kv"]]
    if c["kv"] == "fp8":
        moved += 2 * (keys // PAGE) * c["hk"] * 4
    moved += 2 * sum(new) * c["hq"] * c["d"] * size + keys // PAGE * 4
    return {"bytes": moved, "flops": 4 * pairs * c["hq"] * c["d"]}


# ------------------------------------------------------------------------------- in 64 bits


def exact(case, seed):
    state = prepare(case, seed)
    return exact_attend(state) if case["kind"] == "attend" else exact_append(state)


def exact_attend(s):
    """Sequence by sequence and head by head, the visible keys written out by the definition."""
    c = s["case"]
    tables, cu = s["tables"].cpu(), s["cu"].tolist()
    group = c["hq"] // c["hk"]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device=DEVICE)
    for i, (total, count) in enumerate(zip(s["contexts"].tolist(), s["new"].tolist())):
        start = total - count
        lo = max(0, start - c["window"] + 1)
        keys = torch.tensor([j for j in range(total) if j < c["sinks"] or j >= lo])
        page = tables[i, keys // PAGE].long().to(DEVICE)
        row = (keys % PAGE).to(DEVICE)
        keys = keys.to(DEVICE)
        for r0 in range(0, count, 1024):
            at = torch.arange(start + r0, start + min(count, r0 + 1024), device=DEVICE)[:, None]
            hidden = (keys > at) | ((keys <= at - c["window"]) & (keys >= c["sinks"]))
            rows = slice(cu[i] + r0, cu[i] + r0 + at.shape[0])
            for h in range(c["hk"]):
                k, v = s["k"][page, row, h].double(), s["v"][page, row, h].double()
                if c["kv"] == "fp8":
                    k = k * s["k_scale"][page, h].double()[:, None]
                    v = v * s["v_scale"][page, h].double()[:, None]
                for g in range(h * group, (h + 1) * group):
                    score = s["q"][rows, g].double() @ k.t().contiguous() / math.sqrt(c["d"])
                    score[hidden] = -math.inf
                    out[rows, g] = torch.softmax(score, dim=1) @ v
    return out


def exact_append(s):
    c = s["case"]
    turn = s["positions"]
    cos, sin = s["cos"].double()[turn][:, None], s["sin"].double()[turn][:, None]
    half = c["d"] // 2

    def turned(x):
        x = x.double()
        a, b = x[..., :half], x[..., half:]
        return torch.cat((a * cos[..., :half] - b * sin[..., :half],
                          b * cos[..., half:] + a * sin[..., half:]), dim=-1)

    def written(pool, scale, x):
        slots = s["slots"].tolist()
        if scale is None:
            pool = pool.double()
            flat = pool.view(-1, *pool.shape[2:])
            for t0 in range(0, len(slots), 4096):
                part = [t for t in range(t0, min(len(slots), t0 + 4096)) if slots[t] >= 0]
                flat[torch.tensor([slots[t] for t in part], device=DEVICE)] = x[part]
            return pool
        held = pool.double() * scale.double()[:, None, :, None]
        runs = {}
        for t, slot in enumerate(slots):
            if slot >= 0:
                runs.setdefault(slot // PAGE, []).append((slot % PAGE, t))
        for page, rows in runs.items():
            first, ts = rows[0][0], [t for _, t in rows]
            old = scale[page].double() if first > 0 else torch.zeros_like(scale[page]).double()
            need = torch.exp2(torch.ceil(torch.log2(x[ts].abs().amax(dim=(0, 2)) / E4M3_MAX)))
            size = torch.maximum(old, need)[:, None]
            held[page] = pool[page].double() * size              # (rows behind: their codes stay)
            kept = pool[page, :first].double() * old[:, None]
            held[page, :first] = nearest_e4m3(kept / size) * size
            held[page, first:first + len(ts)] = nearest_e4m3(x[ts] / size) * size
        return held

    return {"q": turned(s["q"]), "k": written(s["k_pool"], s["k_scale"], turned(s["k"])),
            "v": written(s["v_pool"], s["v_scale"], s["v"].double())}


def nearest_e4m3(x):
    """The nearest value with three fraction bits and an exponent of at least -6, ties to even."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return (torch.round(x / step) * step).clamp(-E4M3_MAX, E4M3_MAX)
