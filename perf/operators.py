"""The quantised attention operators as they are measured: attention over packed prompts, attention of new tokens over a paged
cache, the paging plan (block tables and slot maps from request lengths) and the cache write.

Everything is in the fixed point of the graph executor: int32 tensors at scale S = 2^14, products rescaled by a floor shift and
a clamp (the Einsum and Mul nodes), softmax through the two digit tables of SoftmaxLastAxis.  With `own` false the operators are
elementary torch operations; with `own` true they are the framework's entry points (jolt_atlas_amd.attention)."""
import math
import random

import torch

own = False

SCALE_BITS = 14
S = 1 << SCALE_BITS
I32_MIN, I32_MAX = -(1 << 31), (1 << 31) - 1


# ---------------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # nanoGPT's attention: one block of 64 tokens, 4 heads of 16 (latency)
        dict(name="prompt_nano", op="prompt", heads=4, kv_heads=4, dim=16, seqs=1, longest=64, mix=1, fused=True, scaled=True, causal=True),
        # a packed batch of GPT-2 shaped prompts (16 heads of 64), lengths from none to the model's 1024, q / k / v as slices of one c_attn output
        dict(name="prompt_gpt2", op="prompt", heads=16, kv_heads=16, dim=64, seqs=12, longest=1024, mix=2, fused=True, scaled=False, causal=True),
        # odd sizes: 15 heads over 5, head size 80, lengths that no tile divides
        dict(name="prompt_odd", op="prompt", heads=15, kv_heads=5, dim=80, seqs=9, longest=1201, mix=3, fused=False, scaled=True, causal=True),
        # long prompts with grouped heads
        dict(name="prompt_long", op="prompt", heads=32, kv_heads=8, dim=128, seqs=6, longest=6000, mix=4, fused=False, scaled=True, causal=True),
        # one user, one token, GPT-2's context (latency)
        dict(name="cached_one", op="cached", heads=16, kv_heads=16, dim=64, seqs=1, longest=1000, new=1, mix=5, block=16, bits=32, scaled=False, causal=True),
        # a serving step: 64 requests, one token each, ragged contexts
        dict(name="cached_batch", op="cached", heads=32, kv_heads=8, dim=128, seqs=64, longest=8191, new=1, mix=6, block=64, bits=32, scaled=True, causal=True),
        # few long contexts in a 16-bit cache
        dict(name="cached_long16", op="cached", heads=32, kv_heads=4, dim=128, seqs=4, longest=65000, new=1, mix=7, block=128, bits=16, scaled=True, causal=True),
        # chunks of a prompt that continues over a cache, beside single tokens of other requests
        dict(name="cached_chunk", op="cached", heads=32, kv_heads=8, dim=128, seqs=12, longest=5001, new=130, mix=8, block=32, bits=32, scaled=True, causal=True),
        # the serving step's new keys and values go to their slots (latency), and a long prompt's
        dict(name="write_step", op="write", kv_heads=8, dim=128, tokens=64, mix=9, block=64, bits=32),
        dict(name="write_prompt", op="write", kv_heads=8, dim=128, tokens=16001, mix=10, block=64, bits=16),
        # the plan of a serving step, and of a large batch that starts prompts and continues others
        dict(name="plan_step", op="plan", seqs=64, longest=8191, new=1, mix=11, block=64),
        dict(name="plan_many", op="plan", seqs=4000, longest=4001, new=300, mix=12, block=16),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["prompt", "prompt", "cached", "cached", "cached", "write", "plan"])
    mix = rng.randrange(1 << 30)
    kv_heads = rng.choice([1, 2, 4, 5, 8])
    group = rng.choice([1, 1, 2, 3, 4, 8])
    dim = rng.choice([4, 16, 32, 40, 64, 64, 80, 96, 128, 128, 192, 256])
    if op == "plan":
        return dict(op=op, seqs=_log_int(rng, 1, 4000), longest=_log_int(rng, 20, 8000), new=rng.choice([1, 1, 7, 64, 300]), mix=mix, block=rng.choice([1, 16, 32, 64, 128]))
    if op == "write":
        return dict(op=op, kv_heads=kv_heads, dim=dim, tokens=_log_int(rng, 1, 16000), mix=mix, block=rng.choice([1, 16, 32, 64, 128]), bits=rng.choice([16, 32]))
    while True:
        c = dict(op=op, heads=kv_heads * group, kv_heads=kv_heads, dim=dim, mix=mix, scaled=rng.random() < 0.7, causal=rng.random() < 0.8)
        if op == "prompt":
            c.update(seqs=_log_int(rng, 1, 40), longest=_log_int(rng, 1, 6000), fused=rng.random() < 0.5)
        else:
            c.update(seqs=_log_int(rng, 1, 64), longest=_log_int(rng, 10, 40000), new=rng.choice([1, 1, 1, 2, 5, 17, 130]), block=rng.choice([8, 16, 32, 64, 128, 256]), bits=rng.choice([16, 32, 32]))
        w = work(c)
        if w["flops"] <= 2.5e11 and w["bytes"] <= 1.1e9:
            return c


def _prompt_lens(c):
    r = random.Random(c["mix"])
    lens = [c["longest"]] + [_log_int(r, 1, c["longest"]) for _ in range(c["seqs"] - 1)]
    if len(lens) >= 4:                                      # an empty sequence and a single token among the others
        lens[1], lens[2] = 0, 1
    r.shuffle(lens)
    return lens


def _cached_lens(c):
    """(keys of each sequence with the new ones, its new tokens)"""
    r = random.Random(c["mix"])
    keys = [c["longest"]] + [_log_int(r, max(1, c["longest"] // 40), c["longest"]) for _ in range(c["seqs"] - 1)]
    new = [c["new"] if c["new"] == 1 else r.randint(1, c["new"]) for _ in keys]
    new[0] = c["new"]
    if c["new"] > 1 and len(new) >= 4:                      # a request that pauses, one that gets a single token
        new[1], new[2] = 0, 1
    return [max(k, n) for k, n in zip(keys, new)], new


def _plan_lens(c):
    """(tokens in the cache, new tokens; -1: the request has ended and gives its blocks back)"""
    r = random.Random(c["mix"])
    have = [c["longest"]] + [r.choice([0, _log_int(r, 1, c["longest"])]) if c["new"] > 1 else _log_int(r, 1, c["longest"]) for _ in range(c["seqs"] - 1)]
    new = [c["new"] if c["new"] == 1 else _log_int(r, 1, c["new"]) for _ in have]
    for i in range(1, len(new)):
        if r.random() < 0.06:
            new[i] = r.choice([0, -1])
    return have, new


def _blocks(n, b):
    return -(-n // b)


def _pairs(keys, new, causal):
    return sum(n * k - (n * (n - 1) // 2 if causal else 0) for k, n in zip(keys, new))


def work(c):
    if c["op"] == "plan":
        have, new = _plan_lens(c)
        B = c["block"]
        fresh = sum(_blocks(h + n, B) - _blocks(h, B) for h, n in zip(have, new) if n > 0)
        back = sum(_blocks(h, B) for h, n in zip(have, new) if n < 0)
        total = sum(n for n in new if n > 0)
        return {"bytes": 4.0 * (4 * len(have) + 1) + 8.0 * (fresh + back) + 12.0 * total, "flops": 0.0}
    if c["op"] == "write":
        return {"bytes": 2.0 * c["tokens"] * c["kv_heads"] * c["dim"] * (4 + c["bits"] // 8) + 8.0 * c["tokens"], "flops": 0.0}
    if c["op"] == "prompt":
        lens = _prompt_lens(c)
        n, keys, size = sum(lens), sum(lens), 4
        pairs = _pairs(lens, lens, c["causal"])
    else:
        k, new = _cached_lens(c)
        n, keys, size = sum(new), sum(x for x, t in zip(k, new) if t), c["bits"] // 8
        pairs = _pairs(k, new, c["causal"])
    d = c["dim"]
    return {"bytes": 8.0 * n * c["heads"] * d + 2.0 * size * keys * c["kv_heads"] * d, "flops": 4.0 * d * c["heads"] * pairs}


# ------------------------------------------------------------------------------------------------------------- prepare
def _values(g, shape, sigma, limit=(1 << 18) - 1, out=None):
    """activations at scale 2^14: normal, with one channel in 16 four times as large (as projections of trained models have them)"""
    x = torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)
    x[..., ::16] *= 4.0
    return (x * (sigma * S)).round_().clamp_(-limit - 1, limit).to(torch.int32)


def _tables():
    """the two digit tables of exp(-z / S): z = 512 hi + lo"""
    hi = [int(math.floor(S * math.exp(-512.0 * h / S) + 0.5)) for h in range(334)] + [0] * (512 - 334)
    lo = [int(math.floor(S * math.exp(-float(l) / S) + 0.5)) for l in range(512)]
    return torch.tensor(hi, device="cuda"), torch.tensor(lo, device="cuda")


def _score_mul(c):
    return int(round(S / math.sqrt(c["dim"]))) if c["scaled"] else S


def prepare(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": c}
    if own:
        from jolt_atlas_amd import attention
        s["lib"] = attention
    if c["op"] == "plan":
        have, new = _plan_lens(c)
        B, n = c["block"], len(have)
        cols = max(_blocks(h + max(t, 0), B) for h, t in zip(have, new)) + 1
        need = sum(_blocks(h + max(t, 0), B) for h, t in zip(have, new))
        s["n_blocks"] = need + 17
        ids = torch.randperm(s["n_blocks"], generator=g, device="cuda").to(torch.int32)
        table = torch.full((n, cols), -1, dtype=torch.int32, device="cuda")
        used, host = 0, []
        for h in have:
            host.append((used, used + _blocks(h, B)))
            used += _blocks(h, B)
        counts = torch.tensor([b - a for a, b in host], device="cuda")
        table[torch.arange(cols, device="cuda")[None, :] < counts[:, None]] = ids[:used]
        free = torch.zeros(s["n_blocks"], dtype=torch.int32, device="cuda")
        free[: s["n_blocks"] - used] = ids[used:]
        cap = sum(max(t, 0) for t in new) + 5
        s.update(have=torch.tensor(have, dtype=torch.int32, device="cuda"), new=torch.tensor(new, dtype=torch.int32, device="cuda"), table=table, free=free,
                 n_free=torch.tensor([s["n_blocks"] - used], dtype=torch.int32, device="cuda"), n_free_out=torch.zeros(1, dtype=torch.int32, device="cuda"),
                 cu=torch.zeros(n + 1, dtype=torch.int32, device="cuda"), lens=torch.zeros(n, dtype=torch.int32, device="cuda"),
                 slots=torch.zeros(cap, dtype=torch.int64, device="cuda"), positions=torch.zeros(cap, dtype=torch.int32, device="cuda"),
                 status=torch.zeros(1, dtype=torch.int32, device="cuda"))
        if own:
            s["pager"] = attention.Pager(block_size=B, n_blocks=s["n_blocks"])
            s["workspace"] = torch.empty(s["pager"].workspace_bytes(n, cap), dtype=torch.uint8, device="cuda")
        return s
    dtype = torch.int16 if c.get("bits") == 16 else torch.int32
    # what a 16-bit cache holds is below 2.0; elsewhere keys and values have unit size
    sigma, limit = (0.35, 32767) if c.get("bits") == 16 else (1.0, (1 << 18) - 1)
    if c["op"] == "write":
        n, h, d, B = c["tokens"], c["kv_heads"], c["dim"], c["block"]
        n_blocks = 2 * _blocks(n, B) + 3
        perm = torch.randperm(n_blocks * B, generator=g, device="cuda")[:n]
        perm[:: 97] = -1 if n > 97 else perm[::97]          # padding rows of a captured step
        s.update(k=_values(g, (n, h, d), sigma, limit), v=_values(g, (n, h, d), sigma, limit), slots=perm.contiguous(), status=torch.zeros(1, dtype=torch.int32, device="cuda"))
        s["k_cache"] = torch.randint(-99, 99, (n_blocks, h, B, d), generator=g, device="cuda", dtype=dtype)
        s["v_cache"] = torch.randint(-99, 99, (n_blocks, h, B, d), generator=g, device="cuda", dtype=dtype)
        if own:
            s["cache"] = attention.KVCache(s["k_cache"], s["v_cache"])
        return s
    H, KV, d = c["heads"], c["kv_heads"], c["dim"]
    q_sigma = 1.0 if c["scaled"] else 1.5 / math.sqrt(d)
    if c["op"] == "prompt":
        lens = _prompt_lens(c)
        n = sum(lens)
        cu = [0]
        for x in lens:
            cu.append(cu[-1] + x)
        if c["fused"]:                                      # slices of one projection's output
            row = _values(g, (n, H + 2 * KV, d), 1.0)
            row[:, :H] = _values(g, (n, H, d), q_sigma)
            s["q"], s["k"], s["v"] = row[:, :H], row[:, H:H + KV], row[:, H + KV:]
        else:
            s["q"], s["k"], s["v"] = _values(g, (n, H, d), q_sigma), _values(g, (n, KV, d), 1.0), _values(g, (n, KV, d), 1.0)
        s["keys"], s["new"] = lens, lens
    else:
        keys, new = _cached_lens(c)
        B, n = c["block"], sum(new)
        cu = [0]
        for x in new:
            cu.append(cu[-1] + x)
        need = sum(_blocks(k, B) for k in keys)
        n_blocks = need + 3
        ids = torch.randperm(n_blocks, generator=g, device="cuda").to(torch.int32)
        cols = max(_blocks(k, B) for k in keys)
        table = torch.full((len(keys), cols), -1, dtype=torch.int32, device="cuda")
        counts = torch.tensor([_blocks(k, B) for k in keys], device="cuda")
        table[torch.arange(cols, device="cuda")[None, :] < counts[:, None]] = ids[:need]
        s["k_cache"] = _values(g, (n_blocks, KV, B, d), sigma, limit).to(dtype)
        s["v_cache"] = _values(g, (n_blocks, KV, B, d), sigma, limit).to(dtype)
        s["q"] = _values(g, (n, H, d), q_sigma)
        s.update(keys=keys, new=new, table=table, lens=torch.tensor(keys, dtype=torch.int32, device="cuda"))
        if own:
            s["cache"] = attention.KVCache(s["k_cache"], s["v_cache"])
    s["cu"] = torch.tensor(cu, dtype=torch.int32, device="cuda")
    s["out"] = torch.zeros((n, H, d), dtype=torch.int32, device="cuda")
    if own:
        s["attn"] = attention.Attention(H, KV, d, score_mul=_score_mul(c), causal=c["causal"])
        size = s["attn"].prompt_workspace_bytes(len(s["keys"]), n) if c["op"] == "prompt" else s["attn"].cached_workspace_bytes(len(s["keys"]), n, s["cache"], s["table"].shape[1])
        s["workspace"] = torch.empty(size, dtype=torch.uint8, device="cuda")
    else:
        s["tables"] = _tables()
    return s


# ----------------------------------------------------------------------------------------------------------------- run
def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_own(s):
    c, stream = s["case"], torch.cuda.current_stream().cuda_stream
    if c["op"] == "plan":
        s["pager"].plan(s["have"], s["new"], s["table"], s["free"], s["n_free"], s["n_free_out"], s["cu"], s["lens"], s["slots"], s["positions"], s["status"],
                        workspace=s["workspace"], stream=stream)
        return {k: s[k] for k in ("table", "free", "n_free_out", "cu", "lens", "slots", "positions", "status")}
    if c["op"] == "write":
        s["cache"].write(s["k"], s["v"], s["slots"], status=s["status"], stream=stream)
        return {k: s[k] for k in ("k_cache", "v_cache", "status")}
    if c["op"] == "prompt":
        return s["attn"].prompt(s["q"], s["k"], s["v"], s["cu"], s["out"], workspace=s["workspace"], stream=stream)
    return s["attn"].cached(s["q"], s["cu"], s["lens"], s["cache"], s["table"], s["out"], workspace=s["workspace"], stream=stream)


def _run_plain(s):
    c = s["case"]
    if c["op"] == "plan":
        return _plain_plan(s)
    if c["op"] == "write":
        keep = (s["slots"] >= 0).nonzero()[:, 0]
        at, B = s["slots"][keep], c["block"]
        for x, cache in ((s["k"], s["k_cache"]), (s["v"], s["v_cache"])):
            info = torch.iinfo(cache.dtype)
            s["status"] |= ((x[keep] < info.min) | (x[keep] > info.max)).any().to(torch.int32)
            cache[at // B, :, at % B] = x[keep].clamp(info.min, info.max).to(cache.dtype)
        return {k: s[k] for k in ("k_cache", "v_cache", "status")}
    at = 0
    for i, (m, n) in enumerate(zip(s["keys"], s["new"])):
        if n == 0:
            continue
        if c["op"] == "prompt":
            k, v = s["k"][at:at + n], s["v"][at:at + n]
        else:
            ids = s["table"][i, : _blocks(m, c["block"])].long()
            k, v = (x[ids].permute(0, 2, 1, 3).reshape(-1, c["kv_heads"], c["dim"])[:m] for x in (s["k_cache"], s["v_cache"]))
        rows = max(1, (1 << 27) // (c["heads"] * m))        # bounds the score matrix that is held at a time
        for a in range(0, n, rows):
            b = min(n, a + rows)
            s["out"][at + a:at + b] = _plain_attention(s["q"][at + a:at + b], k, v, m - n + a, _score_mul(c), c["causal"], s["tables"])
        at += n
    return s["out"]


def _rescale(x):
    """floor(x / S), clamped to 32 bits; x holds whole numbers in float64 (all sums here stay below 2^53)"""
    return torch.floor(x / S).clamp_(I32_MIN, I32_MAX)


def _plain_attention(q, k, v, first, score_mul, causal, tables):
    """rows of q [n, H, d] over keys [m, KV, d]; row i sees the keys up to first + i"""
    (n, H, d), (m, KV, _) = q.shape, k.shape
    G = H // KV
    qd = q.double().reshape(n, KV, G, d).permute(1, 2, 0, 3).reshape(KV, G * n, d).contiguous()
    kd = k.double().permute(1, 2, 0).contiguous()
    vd = v.double().permute(1, 0, 2).contiguous()
    x = _rescale(_rescale(torch.matmul(qd, kd)) * score_mul).reshape(KV, G, n, m)
    if causal:
        gone = torch.arange(m, device=q.device)[None, :] > first + torch.arange(n, device=q.device)[:, None]
        x.masked_fill_(gone, -math.inf)
    z = (x.amax(dim=-1, keepdim=True) - x).clamp_(max=float((1 << 18) - 1)).to(torch.int32)
    e = (tables[0][z >> 9] * tables[1][z & 511]) >> SCALE_BITS
    if causal:
        e.masked_fill_(gone, 0)
    w = (S * S) // e.sum(dim=-1, keepdim=True)
    p = ((e * w) >> SCALE_BITS).double().reshape(KV, G * n, m)
    y = _rescale(torch.matmul(p, vd)).to(torch.int32)
    return y.reshape(KV, G, n, d).permute(2, 0, 1, 3).reshape(n, H, d)


def _plain_plan(s):
    c, B, dev = s["case"], s["case"]["block"], s["have"].device
    have, new = s["have"].long(), s["new"].long()
    ended = new < 0
    have_blocks = (have + B - 1) // B
    top = s["n_free"].long()
    # the blocks of ended requests go onto the stack, in the order of requests and of their positions
    cols = torch.arange(s["table"].shape[1], device=dev)
    mine = cols[None, :] < have_blocks[:, None]
    back = s["table"][mine & ended[:, None]]
    s["free"][top + torch.arange(back.numel(), device=dev)] = back
    top = top + back.numel()
    n_new = new.clamp(min=0)
    fresh = torch.where(ended, 0, (have + n_new + B - 1) // B - have_blocks)
    start = torch.cumsum(fresh, 0) - fresh
    grows = (cols[None, :] >= have_blocks[:, None]) & (cols[None, :] < (have_blocks + fresh)[:, None])
    order = start[:, None] + cols[None, :] - have_blocks[:, None]
    s["table"][grows] = s["free"][(top - 1 - order)[grows]]
    s["n_free_out"][:] = top - fresh.sum()
    s["cu"][1:] = torch.cumsum(n_new, 0)
    s["lens"][:] = torch.where(ended, 0, have + n_new)
    token = torch.arange(s["slots"].numel(), device=dev)
    seq = torch.searchsorted(s["cu"][1:].contiguous(), token.to(torch.int32), right=True).clamp_(max=have.numel() - 1)
    inside = token < s["cu"][-1]
    pos = torch.where(inside, have[seq] + token - s["cu"][seq], 0)
    block = s["table"][seq, pos // B].long()
    s["slots"][:] = torch.where(inside, block * B + pos % B, -1)
    s["positions"][:] = pos
    return {k: s[k] for k in ("table", "free", "n_free_out", "cu", "lens", "slots", "positions", "status")}


# --------------------------------------------------------------------------------------------------------------- exact
def exact(c, seed):
    """the operators from their definition, in 64-bit integers: products summed one by one, lists walked on the host"""
    global own
    was, own = own, False
    try:
        s = prepare(c, seed)
    finally:
        own = was
    if c["op"] == "plan":
        return _exact_plan(s)
    if c["op"] == "write":
        slots = s["slots"].tolist()
        got = {}
        for name in ("k", "v"):
            cache = s[name + "_cache"].long()
            lo, hi = (-(1 << 15), (1 << 15) - 1) if c["bits"] == 16 else (I32_MIN, I32_MAX)
            flat = cache.permute(0, 2, 1, 3).reshape(-1, c["kv_heads"], c["dim"])
            src = [i for i, t in enumerate(slots) if t >= 0]
            dst = [t for t in slots if t >= 0]
            if src:
                flat.index_copy_(0, torch.tensor(dst, device="cuda"), torch.minimum(torch.maximum(s[name].long(), torch.tensor(lo, device="cuda")), torch.tensor(hi, device="cuda"))[torch.tensor(src, device="cuda")])
            got[name + "_cache"] = flat.reshape(cache.shape[0], c["block"], c["kv_heads"], c["dim"]).permute(0, 2, 1, 3).contiguous()
        got["status"] = torch.zeros(1, dtype=torch.int64)
        return got
    if work(c)["flops"] > 4e11:
        return None
    base = torch.tensor([max(0, round(S * math.exp(-h / 32.0))) for h in range(334)] + [0] * 178, dtype=torch.int64, device="cuda")
    fine = torch.tensor([round(S * math.exp(-l / 16384.0)) for l in range(512)], dtype=torch.int64, device="cuda")
    out = torch.zeros(s["out"].shape, dtype=torch.int64, device="cuda")
    G, mul, row = c["heads"] // c["kv_heads"], _score_mul(c), 0
    for i, (m, n) in enumerate(zip(s["keys"], s["new"])):
        for h in range(c["kv_heads"]) if n else ():
            if c["op"] == "prompt":
                k, v = s["k"][row:row + n, h].long(), s["v"][row:row + n, h].long()
            else:
                pages = s["table"][i].tolist()[: _blocks(m, c["block"])]
                k = torch.cat([s["k_cache"][p, h] for p in pages])[:m].long()
                v = torch.cat([s["v_cache"][p, h] for p in pages])[:m].long()
            kt, vt = k.t().contiguous(), v.t().contiguous()
            step = max(1, (1 << 27) // (m * G))
            for a in range(0, n, step):
                b = min(n, a + step)
                q = s["q"][row + a:row + b, h * G:(h + 1) * G].long()              # [rows, G, d]
                x = torch.zeros((b - a, G, m), dtype=torch.int64, device="cuda")
                for j in range(c["dim"]):
                    x.addcmul_(q[:, :, j, None], kt[j][None, None, :])
                x = (x >> 14).clamp(I32_MIN, I32_MAX)
                x = ((x * mul) >> 14).clamp(I32_MIN, I32_MAX)
                seen = torch.ones((b - a, 1, m), dtype=torch.bool, device="cuda")
                if c["causal"]:
                    seen = (torch.arange(m, device="cuda")[None, :] - torch.arange(a, b, device="cuda")[:, None] <= m - n)[:, None, :]
                z = torch.where(seen, x, torch.tensor(-(1 << 40), device="cuda"))
                z = z.max(dim=2, keepdim=True).values - z
                e = torch.where(seen & (z < (1 << 18)), (base[(z >> 9).clamp(max=511)] * fine[z & 511]) >> 14, 0)
                p = (e * ((1 << 28) // e.sum(dim=2, keepdim=True))) >> 14
                for j in range(c["dim"]):
                    out[row + a:row + b, h * G:(h + 1) * G, j] = ((p * vt[j][None, None, :]).sum(dim=2) >> 14).clamp(I32_MIN, I32_MAX)
        row += n
    return out


def _exact_plan(s):
    c, B = s["case"], s["case"]["block"]
    have, new = s["have"].tolist(), s["new"].tolist()
    table, free = s["table"].cpu().numpy().copy(), s["free"].cpu().numpy().copy()
    top = int(s["n_free"])
    for i, t in enumerate(new):
        if t < 0:
            for b in range(_blocks(have[i], B)):
                free[top] = table[i, b]
                top += 1
    cu, lens, slots, positions = [0], [], [], []
    for i, t in enumerate(new):
        lens.append(0 if t < 0 else have[i] + t)
        for b in range(_blocks(have[i], B), _blocks(lens[-1], B)):
            top -= 1
            table[i, b] = free[top]
        for p in range(have[i], lens[-1]):
            slots.append(int(table[i, p // B]) * B + p % B)
            positions.append(p)
        cu.append(len(slots))
    pad = s["slots"].numel() - len(slots)
    as_int = lambda x: torch.as_tensor(x, dtype=torch.int64)  # noqa: E731
    return {"table": as_int(table), "free": as_int(free), "n_free_out": as_int([top]), "cu": as_int(cu), "lens": as_int(lens), "slots": as_int(slots + [-1] * pad),
            "positions": as_int(positions + [0] * pad), "status": as_int([0])}
