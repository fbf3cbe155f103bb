"""Cases of the rotary and latent-attention operators: what each is measured on.

Geometry: every token keeps one latent vector of ``R`` values and a rotary key of
``P`` = 64 values shared by all heads; a query head has 128 position-free and 64
rotary dims, a value head 128.  ``w`` [H, 256, R] holds each head's key and value
expansions (128 rows each).  Lengths, page tables and page order are ragged and
permuted, as a serving loop leaves them.
"""
import math
import random

import torch

own = False

NOPE, P, V = 128, 64, 128
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # rotary positions: one decode step's query heads (latency), a ragged chunk with the
        # interleaved layout over part of the head, a long fp32 pass over a stretched table
        {"name": "rope_step", "op": "rope", "T": 16, "H": 32, "D": 128, "rot": 64, "offset": 64, "interleaved": True,
         "dtype": "bf16", "max_pos": 32768, "stretch": 1.0},
        {"name": "rope_part", "op": "rope", "T": 2043, "H": 28, "D": 128, "rot": 32, "offset": 0, "interleaved": True,
         "dtype": "fp16", "max_pos": 32768, "stretch": 1.0},
        {"name": "rope_far", "op": "rope", "T": 16384, "H": 64, "D": 128, "rot": 128, "offset": 0,
         "interleaved": False, "dtype": "fp32", "max_pos": 131072, "stretch": 4.0},
        # cache write: one decode step of a batch, one large prefill chunk
        {"name": "write_step", "op": "write", "T": 64, "H": 32, "R": 512, "page": 16, "interleaved": True,
         "max_pos": 32768},
        {"name": "write_chunk", "op": "write", "T": 8191, "H": 128, "R": 512, "page": 16, "interleaved": False,
         "max_pos": 32768},
        # decode: a lone request; a shard with few heads over long contexts (memory); the
        # narrow latent; an ordinary batch with every head; the largest batch
        {"name": "decode_one", "op": "decode", "B": 1, "H": 32, "R": 512, "page": 16, "lo": 1001, "hi": 1001},
        {"name": "decode_long", "op": "decode", "B": 8, "H": 8, "R": 512, "page": 64, "lo": 30000, "hi": 65000},
        {"name": "decode_narrow", "op": "decode", "B": 33, "H": 20, "R": 256, "page": 16, "lo": 1, "hi": 4096},
        {"name": "decode_batch", "op": "decode", "B": 64, "H": 128, "R": 512, "page": 16, "lo": 500, "hi": 4096},
        {"name": "decode_large", "op": "decode", "B": 192, "H": 128, "R": 512, "page": 64, "lo": 4096, "hi": 8192},
        # prefill: short ragged prompts; a long prompt's chunk over its context, every head
        {"name": "prefill_short", "op": "prefill", "q": "17 1 130 300 64", "ctx": "17 900 130 557 64",
         "H": 28, "R": 512, "page": 16},
        {"name": "prefill_chunk", "op": "prefill", "q": "2048 2048 1999 4096", "ctx": "2048 8192 1999 8001",
         "H": 128, "R": 512, "page": 16},
    ]


def _ints(text):
    """A list of lengths kept as text."""
    return [int(v) for v in text.split()]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rope", "write", "decode", "decode", "prefill", "prefill"])
    if op == "rope":
        dt = rng.choice(["bf16", "fp16", "fp32"])
        D = rng.choice([64, 128, 192])
        rot = rng.choice([r for r in (16, 32, 64, 128) if r <= D])
        H = _log_int(rng, 1, 64)
        return {"op": "rope", "T": _log_int(rng, 1, 10000), "H": H, "D": D, "rot": rot,
                "offset": rng.choice([0, D - rot]), "interleaved": rng.random() < 0.5, "dtype": dt,
                "max_pos": rng.choice([4096, 32768, 131072]), "stretch": rng.choice([1.0, 4.0])}
    if op == "write":
        return {"op": "write", "T": _log_int(rng, 1, 8000), "H": _log_int(rng, 1, 128), "R": rng.choice([256, 512]),
                "page": rng.choice([16, 32, 64]), "interleaved": rng.random() < 0.5, "max_pos": 32768}
    if op == "decode":
        B = _log_int(rng, 1, 192)
        hi = _log_int(rng, 16, min(65536, 1150000 // B))
        return {"op": "decode", "B": B, "H": _log_int(rng, 1, 128), "R": rng.choice([256, 512]),
                "page": rng.choice([16, 32, 64]), "lo": rng.randint(1, hi), "hi": hi}
    n = rng.randint(1, 5)
    q = [_log_int(rng, 1, 2048) for _ in range(n)]
    ctx = [a + rng.choice([0, _log_int(rng, 1, 4000)]) for a in q]
    return {"op": "prefill", "q": " ".join(map(str, q)), "ctx": " ".join(map(str, ctx)),
            "H": _log_int(rng, 1, 128), "R": rng.choice([256, 512]), "page": rng.choice([16, 32, 64])}


# ------------------------------------------------------------------------- inputs
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(g, *shape, dtype=torch.bfloat16, std=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)


def _table(max_pos, rot, stretch):
    """[max_pos, rot] cos | sin of position / stretch, angles in 64 bits."""
    inv = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot)
    a = torch.outer(torch.arange(max_pos, dtype=torch.float64, device="cuda") / stretch, inv)
    return torch.cat([a.cos(), a.sin()], 1).float()


def _pages(g, lens, page):
    """Block tables (int32 [B, max blocks]) of permuted pages, and the number of pages."""
    need = [max(1, -(-n // page)) for n in lens]
    total = sum(need) + 3
    order = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
    bt = torch.zeros(len(lens), max(need), dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(need):
        bt[i, :n] = order[at:at + n]
        at += n
    return bt, total


def _decode_lens(case, seed):
    r = random.Random(seed)
    return [r.randint(case["lo"], case["hi"]) for _ in range(case["B"])]


def prepare(case, seed):
    g = _gen(seed)
    s = {"case": case}
    op = case["op"]
    if op == "rope":
        s["x"] = _randn(g, case["T"], case["H"], case["D"], dtype=DTYPES[case["dtype"]])
        s["pos"] = torch.randint(0, case["max_pos"], (case["T"],), generator=g, device="cuda", dtype=torch.int32)
        s["cs"] = _table(case["max_pos"], case["rot"], case["stretch"])
        s["out"] = torch.empty_like(s["x"])
        return s
    R, page, H = case["R"], case["page"], case["H"]
    if op == "write":
        T = case["T"]
        s["q"] = _randn(g, T, H, NOPE + P)[:, :, NOPE:]  # the rotary part of the query heads
        s["kv"] = _randn(g, T, R + P, std=2.0)
        s["w"] = (1.0 + 0.1 * torch.randn(R, generator=g, device="cuda")).to(torch.bfloat16)
        s["pos"] = torch.randint(0, case["max_pos"], (T,), generator=g, device="cuda", dtype=torch.int32)
        s["cs"] = _table(case["max_pos"], P, 1.0)
        blocks = -(-T // page) + 2
        s["cache"] = torch.zeros(blocks, page, R + P, dtype=torch.bfloat16, device="cuda")
        s["slots"] = torch.randperm(blocks * page, generator=g, device="cuda")[:T].contiguous()
        s["slots"][T // 2:T // 2 + 1] = -1 if T > 1 else 0  # a padded row writes nothing
        s["q_out"] = torch.empty(T, H, P, dtype=torch.bfloat16, device="cuda")
        return s
    if op == "decode":
        lens = _decode_lens(case, seed)
        rows = case["B"]
    else:
        lens = _ints(case["ctx"])
        rows = sum(_ints(case["q"]))
    bt, total = _pages(g, lens, page)
    s["lens"], s["bt"] = lens, bt
    s["cache"] = _randn(g, total, page, R + P)
    s["q"] = _randn(g, rows, H * (NOPE + P), std=1.5)
    s["w"] = _randn(g, H, NOPE + V, R, std=1.0 / math.sqrt(R))
    s["scale"] = 1.0 / math.sqrt(NOPE + P)
    s["out"] = torch.empty(rows, H * V, dtype=torch.bfloat16, device="cuda")
    s["ctx"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    if own and op == "prefill":
        from kapsl_sdk_b200 import ops

        s["plan"] = ops.latent_prefill_plan(_ints(case["q"]), lens, device="cuda")
    return s


# ------------------------------------------------------------- the framework's calls
def _run_own(s):
    from kapsl_sdk_b200 import ops

    case, op = s["case"], s["case"]["op"]
    if op == "rope":
        return ops.rope(s["x"], s["pos"], s["cs"], offset=case["offset"], interleaved=case["interleaved"],
                        out=s["out"])
    if op == "write":
        ops.rope_latent_write(s["q"], s["kv"], s["pos"], s["slots"], s["cs"], s["w"], 1e-6, s["cache"],
                              interleaved=case["interleaved"], q_out=s["q_out"])
        return [s["q_out"], s["cache"]]
    if op == "decode":
        return ops.latent_decode_attention(s["q"], s["cache"], s["w"], s["bt"], s["ctx"], case["H"],
                                           scale=s["scale"], out=s["out"], max_ctx=max(s["lens"]))
    return ops.latent_prefill_attention(s["q"], s["cache"], s["w"], s["plan"], s["bt"], case["H"], scale=s["scale"],
                                        out=s["out"])


# ----------------------------------------------------------------- the plain forms
def _rotate(x, cs, interleaved):
    """x [T, H, rot], cs [T, rot] in x's type."""
    half = x.shape[-1] // 2
    c, n = cs[:, None, :half], cs[:, None, half:]
    if interleaved:
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack([a * c - b * n, b * c + a * n], -1).reshape(x.shape)
    a, b = x[..., :half], x[..., half:]
    return torch.cat([a * c - b * n, b * c + a * n], -1)


def _rows(s, i, n):
    """The first n cache rows of sequence i."""
    page = s["case"]["page"]
    pages = s["bt"][i, :-(-n // page)].long()
    return s["cache"][pages].reshape(-1, s["cache"].shape[2])[:n]


def run(state):
    if own:
        return _run_own(state)
    s, case, op = state, state["case"], state["case"]["op"]
    if op == "rope":
        x, o, r = s["x"], case["offset"], case["rot"]
        y = _rotate(x[..., o:o + r].float(), s["cs"][s["pos"].long()], case["interleaved"])
        out = s["out"]
        out.copy_(x)
        out[..., o:o + r] = y.to(x.dtype)
        return out
    R, H = case["R"], case["H"]
    if op == "write":
        cs = s["cs"][s["pos"].long()]
        s["q_out"].copy_(_rotate(s["q"].float(), cs, case["interleaved"]))
        kv = s["kv"].float()
        c = kv[:, :R]
        c = c * torch.rsqrt(c.pow(2).mean(-1, keepdim=True) + 1e-6) * s["w"].float()
        row = torch.cat([c, _rotate(kv[:, None, R:], cs, case["interleaved"])[:, 0]], -1).to(torch.bfloat16)
        keep = torch.where(s["slots"] >= 0, s["slots"], s["slots"].max())
        row = torch.where((s["slots"] >= 0)[:, None], row, row[s["slots"].argmax()][None])
        s["cache"].view(-1, R + P)[keep] = row
        return [s["q_out"], s["cache"]]
    q = s["q"].view(-1, H, NOPE + P)
    w = s["w"].float()
    if op == "decode":
        qf = q.float()
        qa = torch.cat([torch.einsum("bhd,hdr->bhr", qf[..., :NOPE], w[:, :NOPE]), qf[..., NOPE:]], -1)
        o = torch.empty(len(s["lens"]), H, R, device="cuda")
        for i, n in enumerate(s["lens"]):
            c = _rows(s, i, n).float()
            p = torch.softmax(qa[i] @ c.T * s["scale"], -1)
            o[i] = p @ c[:, :R]
        s["out"].copy_(torch.einsum("bhr,hvr->bhv", o, w[:, NOPE:]).reshape(-1, H * V))
        return s["out"]
    at = 0
    out = s["out"].view(-1, H, V)
    for i, (n, ctx) in enumerate(zip(_ints(case["q"]), s["lens"])):
        c = _rows(s, i, ctx).float()
        hide = torch.arange(ctx, device="cuda")[None] > torch.arange(ctx - n, ctx, device="cuda")[:, None]
        for h in range(H):
            kv = c[:, :R] @ w[h].T
            k = torch.cat([kv[:, :NOPE], c[:, R:]], -1)
            x = (q[at:at + n, h].float() @ k.T * s["scale"]).masked_fill_(hide, float("-inf"))
            out[at:at + n, h] = (torch.softmax(x, -1) @ kv[:, NOPE:]).to(torch.bfloat16)
        at += n
    return s["out"]


# --------------------------------------------------------------------- 64-bit results
def _turn64(v, table_rows, interleaved):
    """Each pair of v as a complex number times cos + i sin."""
    half = v.shape[-1] // 2
    t = table_rows.double()
    z = torch.complex(t[..., :half], t[..., half:])
    v = v.double()
    if interleaved:
        u = torch.view_as_complex(v.reshape(*v.shape[:-1], half, 2).contiguous())
        return torch.view_as_real(u * z).reshape(v.shape)
    u = torch.complex(v[..., :half], v[..., half:]) * z
    return torch.cat([u.real, u.imag], -1)


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "rope":
        o, r = case["offset"], case["rot"]
        y = s["x"].double()
        y[..., o:o + r] = _turn64(s["x"][..., o:o + r], s["cs"][s["pos"].long()].unsqueeze(1), case["interleaved"])
        return y
    R, H = case["R"], case["H"]
    if op == "write":
        t = s["cs"][s["pos"].long()]
        q = _turn64(s["q"], t.unsqueeze(1), case["interleaved"])
        lat = s["kv"][:, :R].double()
        lat = lat / (lat.square().sum(1, keepdim=True) / R + 1e-6).sqrt() * s["w"].double()
        key = _turn64(s["kv"][:, R:], t, case["interleaved"])
        cache = s["cache"].double().reshape(-1, R + P)
        used = (s["slots"] >= 0).nonzero().flatten()
        cache[s["slots"][used]] = torch.cat([lat, key], 1)[used]
        return [q, cache.view(s["cache"].shape)]
    w = s["w"].double()
    q = s["q"].double().view(-1, H, NOPE + P)
    page = case["page"]
    out = torch.zeros(q.shape[0], H, V, dtype=torch.float64, device="cuda")
    news = [1] * len(s["lens"]) if op == "decode" else _ints(case["q"])
    at = 0
    for i, n in enumerate(news):
        ctx = s["lens"][i]
        idx = torch.arange(ctx, device="cuda")
        c = s["cache"][s["bt"][i, idx // page].long(), idx % page].double()
        if op == "decode":  # the key product moved to the query's side: the same sum in another order
            z = torch.cat([torch.bmm(w[:, :NOPE].transpose(1, 2), q[at][:, :NOPE, None])[..., 0], q[at][:, NOPE:]], 1)
            e = (c @ z.T) * s["scale"]
            e = torch.exp(e - e.max(0).values)
            lat = (e / e.sum(0)).T @ c[:, :R]
            out[at] = torch.bmm(w[:, NOPE:], lat[..., None])[..., 0]
        else:
            seen = idx[None, :] <= (ctx - n + torch.arange(n, device="cuda"))[:, None]
            for h in range(H):
                x = (q[at:at + n, h, :NOPE] @ (c[:, :R] @ w[h, :NOPE].T).T + q[at:at + n, h, NOPE:] @ c[:, R:].T)
                x = torch.where(seen, x * s["scale"], -math.inf)
                e = torch.exp(x - x.max(1, keepdim=True).values)
                out[at:at + n, h] = (e @ (c[:, :R] @ w[h, NOPE:].T)) / e.sum(1, keepdim=True)
        at += n
    return out.view(-1, H * V)


# ------------------------------------------------------------------------------- work
def work(case):
    op, H = case["op"], case["H"]
    if op == "rope":
        n = case["T"] * case["H"] * case["D"]
        size = 4 if case["dtype"] == "fp32" else 2
        return {"bytes": 2 * n * size + case["T"] * (case["rot"] * 4 + 4),
                "flops": 3 * case["T"] * case["H"] * case["rot"]}
    R = case["R"]
    if op == "write":
        T = case["T"]
        return {"bytes": T * (2 * H * P * 2 + 2 * (R + P) * 2 + P * 4 + 12) + R * 2,
                "flops": T * (3 * H * P + 4 * R + 3 * P)}
    weights = H * (NOPE + V) * R * 2
    if op == "decode":
        B, mean = case["B"], (case["lo"] + case["hi"]) / 2
        toks = B * mean
        return {"bytes": int(toks * (R + P) * 2 + weights + B * H * (NOPE + P + V) * 2 + toks / case["page"] * 4),
                "flops": int(toks * H * 2 * (2 * R + P) + 2 * B * H * (NOPE + V) * R)}
    news, lens = _ints(case["q"]), _ints(case["ctx"])
    rows, ctx = sum(news), sum(lens)
    pairs = sum(n * c - n * (n - 1) // 2 for n, c in zip(news, lens))
    return {"bytes": ctx * (R + P) * 2 + weights + rows * H * (NOPE + P + V) * 2,
            "flops": 2 * H * (ctx * (NOPE + V) * R + pairs * (NOPE + P + V))}
