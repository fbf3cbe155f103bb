"""Rotary positions, the latent cache write and both forms of latent attention against
plain 64-bit implementations.

Tolerances.  A rounding to a type with unit u = eps / 2 errs by at most u relative, and as
the errors of many roundings are independent and spread over [-u, u], each counts with a
standard deviation of at most u / sqrt(3).  For attention the test carries the
variance of every rounding that the kernels make (listed at each oracle) to the
output in 64 bits and allows 8 standard deviations: an error of the kernel's own, a
key too many or too few, a wrong page or a wrong weight is far outside.
fp32 sums of up to 600 terms err by at most 600 * 2^-24 < 2^-14 of the terms' absolute sum.
"""
import math
import random

import pytest
import torch

pytestmark = pytest.mark.gpu

U = torch.finfo(torch.bfloat16).eps / 2
F32 = 2.0 ** -14
NAN = float("nan")


@pytest.fixture(scope="module")
def dev():
    from kapsl_sdk_b200._ext import cuda_ops

    cuda_ops()
    return torch.device("cuda", 0)


def within(got, exp, tol):
    err = (got.double() - exp).abs()
    assert torch.isfinite(got.double()).all()
    bad = int((err > tol).sum())
    worst = float((err / tol.clamp_min(1e-30)).max()) if err.numel() else 0.0
    assert bad == 0, f"{bad} values off, worst {worst:.3g} x"


def no_error(dev):
    from kapsl_sdk_b200 import ops

    torch.cuda.synchronize()
    assert ops.check_errors(dev) == 0


# ------------------------------------------------------------------------------ rope
def rope64(x, pos, cs, offset, interleaved):
    y = x.double().clone()
    P = cs.shape[1]
    v = y[..., offset:offset + P]
    c, s = cs[pos.long()].double()[:, None, :P // 2], cs[pos.long()].double()[:, None, P // 2:]
    a, b = (v[..., 0::2], v[..., 1::2]) if interleaved else (v[..., :P // 2], v[..., P // 2:])
    ya, yb = a * c - b * s, b * c + a * s
    mag = a.abs() + b.abs()
    y[..., offset:offset + P] = torch.stack([ya, yb], -1).flatten(-2) if interleaved else torch.cat([ya, yb], -1)
    m = torch.zeros_like(y)
    m[..., offset:offset + P] = torch.stack([mag, mag], -1).flatten(-2) if interleaved else torch.cat([mag, mag], -1)
    return y, m


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("T,H,D,P,offset", [(1, 1, 64, 64, 0), (5, 3, 192, 64, 128), (130, 28, 128, 32, 0),
                                            (33, 7, 80, 16, 40), (9, 2, 37, 10, 5), (3, 5, 7, 2, 5), (2, 1, 2, 2, 0),
                                            (17, 4, 256, 256, 0), (40, 1, 96, 24, 8)])
def test_rope(dev, dtype, interleaved, T, H, D, P, offset):
    """One rounding (u |y|) and two fp32 products and a sum (3 * 2^-24 of |a| + |b|).  Below the
    smallest normal number t the values are t * eps apart whatever their size, so a rounding
    there errs by up to t * eps / 2 = t * u (fp16: 2^-14 * 2^-11 = 2^-25)."""
    from kapsl_sdk_b200 import ops
    from kapsl_sdk_b200.ops import reference as ref

    g = torch.Generator(device=dev).manual_seed(T * 31 + D)
    u = torch.finfo(dtype).eps / 2
    cs = ref.rope_cos_sin(500, P, 1e4, device=dev,
                          scaling={"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 100})
    pos = torch.randint(0, 500, (T,), generator=g, device=dev, dtype=torch.int32)
    x = torch.randn(T, H, D, generator=g, device=dev).to(dtype)
    exp, mag = rope64(x, pos, cs, offset, interleaved)
    tol = u * exp.abs().clamp_min(torch.finfo(dtype).tiny) + 4 * 2.0 ** -24 * mag
    keep = x.clone()
    within(ops.rope(x, pos, cs, offset, interleaved), exp, tol)
    assert torch.equal(x, keep)
    # a strided view of a wider buffer, in place: nothing else moves
    wide = torch.randn(T, H + 1, D + 3, generator=g, device=dev).to(dtype)
    view = wide[:, 1:, 2:D + 2]
    view.copy_(x)
    before = wide.clone()
    assert ops.rope(view, pos, cs, offset, interleaved, out=view) is view
    within(view, exp, tol)
    before[:, 1:, 2:D + 2] = view
    assert torch.equal(wide, before)
    # heads and tokens swapped in memory, into a strided out
    xt = x.transpose(0, 1).contiguous().transpose(0, 1)
    out = torch.full((T, H, D + 5), 7.0, device=dev, dtype=dtype)
    ops.rope(xt, pos, cs, offset, interleaved, out=out[..., :D])
    within(out[..., :D], exp, tol)
    assert bool((out[..., D:] == 7.0).all())
    # one head shared by all (expanded)
    e = x[:, :1].expand(T, H, D)
    within(ops.rope(e, pos, cs, offset, interleaved), rope64(e, pos, cs, offset, interleaved)[0],
           u * 2 * e.abs().amax() + 1e-5)
    no_error(dev)


@pytest.mark.parametrize("interleaved,P,offset", [(False, 128, 0), (True, 64, 64)])
def test_rope_of_a_prompt(dev, interleaved, P, offset):
    """The served type at a prompt's size, in place and into another buffer."""
    from kapsl_sdk_b200 import ops
    from kapsl_sdk_b200.ops import reference as ref

    T, H, D = 6001, 40, 128
    g = torch.Generator(device=dev).manual_seed(1)
    cs = ref.rope_cos_sin(8192, P, 1e4, device=dev)
    pos = torch.arange(1000, 1000 + T, device=dev, dtype=torch.int32)
    x = torch.randn(T, H, D, generator=g, device=dev).to(torch.bfloat16)
    out = ops.rope(x, pos, cs, offset, interleaved)
    for t0 in range(0, T, 1500):
        part = slice(t0, t0 + 1500)
        exp, mag = rope64(x[part], pos[part], cs, offset, interleaved)
        within(out[part], exp, U * exp.abs() + 4 * 2.0 ** -24 * mag)
    assert torch.equal(ops.rope(x, pos, cs, offset, interleaved, out=x), out)
    no_error(dev)


def test_rope_empty_and_positions_outside(dev):
    from kapsl_sdk_b200 import ops
    from kapsl_sdk_b200.ops import reference as ref

    cs = ref.rope_cos_sin(10, 32, 1e4, device=dev)
    x = torch.randn(4, 2, 64, device=dev, dtype=torch.bfloat16)
    assert ops.rope(x[:0], torch.zeros(0, dtype=torch.int32, device=dev), cs).shape == (0, 2, 64)
    assert ops.rope(x[:, :0], torch.zeros(4, dtype=torch.int32, device=dev), cs).shape == (4, 0, 64)
    pos = torch.tensor([3, 10, -1, 9], device=dev, dtype=torch.int32)
    y = ops.rope(x, pos, cs)
    torch.cuda.synchronize()
    assert ops.check_errors(dev) == 80 and "position" in ops.describe_error(80)
    assert torch.equal(y[1:3], x[1:3]) and not torch.equal(y[0], x[0]) and not torch.equal(y[3], x[3])


def test_rope_refuses(dev):
    from kapsl_sdk_b200 import ops
    from kapsl_sdk_b200.ops import reference as ref

    cs = ref.rope_cos_sin(10, 32, 1e4, device=dev)
    x = torch.randn(4, 2, 64, device=dev, dtype=torch.bfloat16)
    pos = torch.zeros(4, dtype=torch.int32, device=dev)
    for bad in (lambda: ops.rope(x.cpu(), pos, cs), lambda: ops.rope(x.double(), pos, cs),
                lambda: ops.rope(x, pos.long(), cs), lambda: ops.rope(x, pos[:3], cs),
                lambda: ops.rope(x, pos.cpu(), cs),
                lambda: ops.rope(x, pos, cs, offset=33), lambda: ops.rope(x, pos, cs, offset=-1),
                lambda: ops.rope(x, pos, cs[:, :31]), lambda: ops.rope(x, pos, cs.half()),
                lambda: ops.rope(x[0], pos, cs), lambda: ops.rope(x.transpose(1, 2), pos, cs),
                lambda: ops.rope(x, pos, cs, out=torch.empty_like(x[:3])),
                lambda: ops.rope(x, pos, cs, out=torch.empty_like(x.float())),
                lambda: ops.rope(x[:, :, :32], pos, cs, out=x[:, :, 16:48]),
                lambda: ops.rope(x, pos, cs, out=x[:1].expand(4, 2, 64)),
                lambda: ops.rope(x[:, :1].expand(4, 2, 64), pos, cs, out=x[:, :1].expand(4, 2, 64))):
        with pytest.raises((RuntimeError, TypeError)):
            bad()
    no_error(dev)


# ------------------------------------------------------------------------ cache write
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("T,H,R,page", [(1, 1, 512, 16), (7, 28, 512, 16), (130, 128, 256, 32), (65, 3, 512, 64),
                                        (300, 20, 256, 16)])
def test_rope_latent_write(dev, interleaved, T, H, R, page):
    """Latents: one rounding of x * inv * w in fp32 (the mean of R squares errs by less than
    (R / 32 + 5) 2^-24, rsqrt and three products by 2^-21 in all); keys as in test_rope."""
    from kapsl_sdk_b200 import ops
    from kapsl_sdk_b200.ops import reference as ref

    g = torch.Generator(device=dev).manual_seed(T + R)

    def rn(*s):
        return torch.randn(*s, generator=g, device=dev).to(torch.bfloat16)

    cs = ref.rope_cos_sin(700, 64, 1e4, device=dev)
    pos = torch.randint(0, 700, (T,), generator=g, device=dev, dtype=torch.int32)
    blocks = T // page + 3
    slots = torch.randperm(blocks * page, generator=g, device=dev)[:T].contiguous()
    if T > 4:
        slots[2] = -1
    cache = rn(blocks, page, R + 64)
    q, kvw, w = rn(T, H, 192), rn(T, R + 64 + 8), rn(R)
    kv = kvw[:, :R + 64]
    kv[0] = 0  # a row of zeros stays finite
    before, q0 = cache.clone(), q.clone()
    c = kv[:, :R].double()
    lat = c / (c.pow(2).mean(1, keepdim=True) + 1e-6).sqrt() * w.double()
    key, kmag = rope64(kv[:, None, R:], pos, cs, 0, interleaved)
    q_exp, q_mag = rope64(q[..., 128:], pos, cs, 0, interleaved)
    exp = torch.cat([lat, key[:, 0]], 1)
    tol = torch.cat([lat.abs() * (U + 2.0 ** -18), U * key[:, 0].abs() + 2.0 ** -22 * kmag[:, 0]], 1)
    q_tol = U * q_exp.abs() + 2.0 ** -22 * q_mag
    q_out = torch.full((T, H, 72), 5.0, device=dev, dtype=torch.bfloat16)
    ops.rope_latent_write(q[..., 128:], kv, pos, slots, cs, w, 1e-6, cache, interleaved, q_out=q_out[..., :64])
    assert torch.equal(q, q0) and bool((q_out[..., 64:] == 5.0).all())
    within(q_out[..., :64], q_exp, q_tol)
    used = (slots >= 0).nonzero().flatten()
    flat = cache.view(-1, R + 64)
    within(flat[slots[used]], exp[used], tol[used])
    flat[slots[used]] = before.view(-1, R + 64)[slots[used]]
    assert torch.equal(cache, before)  # other rows as they were
    ops.rope_latent_write(q[..., 128:], kv, pos, slots, cs, w, 1e-6, cache, interleaved)
    within(q[..., 128:], q_exp, q_tol)
    assert torch.equal(q[..., :128], q0[..., :128])
    no_error(dev)


def test_rope_latent_write_bounds_and_refusals(dev):
    from kapsl_sdk_b200 import ops
    from kapsl_sdk_b200.ops import reference as ref

    def z(*s, dt=torch.bfloat16):
        return torch.zeros(*s, device=dev, dtype=dt)

    cs = ref.rope_cos_sin(10, 64, 1e4, device=dev)
    cache, w = z(2, 16, 576), z(512) + 1
    q = torch.randn(3, 2, 64, device=dev).to(torch.bfloat16)
    kv, pos = z(3, 576) + 1, z(3, dt=torch.int32)
    slots = torch.tensor([0, 32, 31], device=dev)  # 32 rows: the second lies outside
    ops.rope_latent_write(q, kv, pos, slots, cs, w, 1e-6, cache)
    torch.cuda.synchronize()
    assert ops.check_errors(dev) == 81
    assert bool((cache.view(32, 576)[[0, 31]] != 0).all()) and bool((cache.view(32, 576)[1:31] == 0).all())
    ops.rope_latent_write(q[:0], kv[:0], pos[:0], slots[:0], cs, w, 1e-6, cache)
    bad = [dict(q=z(3, 2, 32)), dict(q=q.float()), dict(kv=z(3, 575)), dict(kv=z(2, 576)), dict(kv=z(3, 576).float()),
           dict(cache=z(2, 16, 448)), dict(cache=z(2, 8, 576)), dict(cache=z(2, 16, 640)[..., :576]), dict(w=z(256)),
           dict(slots=slots.int()), dict(slots=slots[:2]), dict(pos=pos[:2]), dict(cs=cs[:, :32].contiguous()),
           dict(q_out=z(3, 1, 64)), dict(q_out=z(3, 2, 65)[..., :64]), dict(kv=cache.view(32, 576)[:3])]
    for kw in bad:
        a = dict(q=q, kv=kv, pos=pos, slots=slots, cs=cs, w=w, cache=cache, q_out=None)
        a.update(kw)
        with pytest.raises((RuntimeError, TypeError)):
            ops.rope_latent_write(a["q"], a["kv"], a["pos"], a["slots"], a["cs"], a["w"], 1e-6, a["cache"],
                                  q_out=a["q_out"])
    no_error(dev)


@pytest.mark.parametrize("interleaved", [False, True])
def test_tables_without_rows(dev, interleaved):
    """No position lies in an empty table: nothing is read from it, nothing is rotated, the error is recorded."""
    from kapsl_sdk_b200 import ops

    cs = torch.empty(0, 64, device=dev)
    x = torch.randn(5, 3, 64, device=dev).to(torch.bfloat16)
    pos = torch.tensor([0, 1, -1, 5, 7], dtype=torch.int32, device=dev)
    assert torch.equal(ops.rope(x, pos, cs, interleaved=interleaved), x)
    torch.cuda.synchronize()
    assert ops.check_errors(dev) == 80
    cache = torch.zeros(1, 16, 320, device=dev, dtype=torch.bfloat16)
    kv, w = torch.randn(5, 320, device=dev).to(torch.bfloat16), torch.ones(256, device=dev, dtype=torch.bfloat16)
    q = ops.rope_latent_write(x, kv, pos, torch.arange(5, device=dev), cs, w, 1e-6, cache, interleaved,
                              q_out=torch.empty_like(x))
    torch.cuda.synchronize()
    assert ops.check_errors(dev) == 80
    assert torch.equal(q, x) and torch.equal(cache[0, :5, 256:], kv[:, 256:])
    ops.rope_latent_write(x[:0], kv[:0], pos[:0], torch.arange(0, device=dev), cs, w, 1e-6, cache, interleaved)
    no_error(dev)


def test_write_padded_rows_need_no_position(dev):
    """A row whose slot is negative writes nothing and records nothing, whatever its position says; its query
    heads stay as they were."""
    from kapsl_sdk_b200 import ops
    from kapsl_sdk_b200.ops import reference as ref

    cs = ref.rope_cos_sin(10, 64, 1e4, device=dev)
    cache = torch.full((1, 16, 576), 3.0, device=dev, dtype=torch.bfloat16)
    q = torch.randn(4, 2, 64, device=dev).to(torch.bfloat16)
    kv, w = torch.randn(4, 576, device=dev).to(torch.bfloat16), torch.ones(512, device=dev, dtype=torch.bfloat16)
    pos = torch.tensor([5, -1, 10, 2 ** 31 - 1], dtype=torch.int32, device=dev)
    slots = torch.tensor([0, -1, -1, -7], device=dev)
    out = ops.rope_latent_write(q, kv, pos, slots, cs, w, 1e-6, cache, q_out=torch.empty_like(q))
    no_error(dev)
    assert torch.equal(out[1:], q[1:]) and not torch.equal(out[0], q[0])
    assert bool((cache[0, 1:] == 3.0).all()) and not bool((cache[0, 0] == 3.0).any())
    slots[1] = 1  # a row that is written has to have one
    ops.rope_latent_write(q, kv, pos, slots, cs, w, 1e-6, cache, q_out=out)
    torch.cuda.synchronize()
    assert ops.check_errors(dev) == 80


def test_refuses_outputs_that_overlap_themselves(dev):
    """Rows or heads of an output that share memory would be written by several threads."""
    from kapsl_sdk_b200 import ops
    from kapsl_sdk_b200.ops import reference as ref

    cs = ref.rope_cos_sin(10, 64, 1e4, device=dev)
    pos = torch.zeros(4, dtype=torch.int32, device=dev)
    flat = torch.randn(4096, device=dev).to(torch.bfloat16)
    x = torch.randn(4, 3, 64, device=dev).to(torch.bfloat16)
    k = Cache(dev, [40, 50], 512, 16, 3)
    q, w = k.randn(2, 5 * 192), k.randn(5, 256, 512, std=0.04)
    plan = ops.latent_prefill_plan([1, 1], [40, 50], dev)
    kv, nw, slots = k.randn(4, 576), k.randn(512), torch.arange(4, device=dev)
    shared = flat.as_strided((4, 3, 64), (64, 64, 1))  # a token's second head is the next one's first
    rows = flat.as_strided((2, 640), (320, 1))
    before = flat.clone()
    for bad in (lambda: ops.rope(x, pos, cs, out=shared), lambda: ops.rope(shared, pos, cs, out=shared),
                lambda: ops.rope(x, pos, cs, out=flat.as_strided((4, 3, 64), (192, 32, 1))),
                lambda: ops.rope_latent_write(shared, kv, pos, slots, cs, nw, 1e-6, k.cache),
                lambda: ops.rope_latent_write(x, kv, pos, slots, cs, nw, 1e-6, k.cache, q_out=shared),
                lambda: ops.latent_decode_attention(q, k.cache, w, k.bt, k.ctx, 5, out=rows),
                lambda: ops.latent_prefill_attention(q, k.cache, w, plan, k.bt, 5, out=rows)):
        with pytest.raises(RuntimeError):
            bad()
    # heads outside tokens, and tokens outside heads, are both in order; so is reading shared memory
    good = torch.empty(3, 4, 64, device=dev, dtype=torch.bfloat16).transpose(0, 1)
    assert torch.equal(ops.rope(x, pos, cs, out=good), ops.rope(x, pos, cs))
    assert torch.equal(ops.rope(shared, pos, cs), ops.rope(shared.clone(), pos, cs))
    no_error(dev)
    assert torch.equal(flat, before)


def test_write_reads_a_weight_just_written(dev):
    """The norm weight may come from the kernel right before, which lets the write kernel start early."""
    from kapsl_sdk_b200 import ops
    from kapsl_sdk_b200.ops import reference as ref

    R, T = 512, 2000
    cs = ref.rope_cos_sin(10, 64, 1e4, device=dev)
    pos, slots = torch.zeros(T, dtype=torch.int32, device=dev), torch.arange(T, device=dev)
    kv = torch.ones(T, R + 64, device=dev, dtype=torch.bfloat16)  # normed: 1 / sqrt(1 + eps) = 1
    q = torch.zeros(T, 1, 64, device=dev, dtype=torch.bfloat16)
    w = torch.zeros(1, R, device=dev, dtype=torch.bfloat16)
    # silu(30) = 30 to a part in 2^43, times 2^i
    xs = [torch.cat([torch.full((1, R), 30.0), torch.full((1, R), 2.0 ** i)], 1).to(torch.bfloat16).to(dev) for i in range(8)]
    caches = [torch.zeros(125, 16, R + 64, device=dev, dtype=torch.bfloat16) for _ in range(8)]
    for _ in range(20):
        torch.cuda.synchronize()
        for x, cache in zip(xs, caches):
            ops.silu_mul(x, out=w)
            ops.rope_latent_write(q, kv, pos, slots, cs, w[0], 0.0, cache)
        torch.cuda.synchronize()
        for i, cache in enumerate(caches):
            assert bool((cache[..., :R] == 30.0 * 2.0 ** i).all())
            cache.zero_()
    no_error(dev)


def test_write_refuses_latents_that_its_queries_overwrite(dev):
    """In one projection's rows the latents may lie before or behind the heads, not among them."""
    from kapsl_sdk_b200 import ops
    from kapsl_sdk_b200.ops import reference as ref

    T, H, R = 5, 2, 256
    cs = ref.rope_cos_sin(10, 64, 1e4, device=dev)
    pos, slots = torch.arange(T, dtype=torch.int32, device=dev), torch.arange(T, device=dev)
    cache = torch.zeros(1, 16, R + 64, dtype=torch.bfloat16, device=dev)
    w = torch.ones(R, dtype=torch.bfloat16, device=dev)
    y = torch.randn(T, 2 * (R + 64) + H * 192, device=dev).to(torch.bfloat16)
    q = y[:, R + 64:R + 64 + H * 192].view(T, H, 192)[..., 128:]
    for at in (0, R + 64 + H * 192):
        for n in (T, 1):
            ops.rope_latent_write(q[:n], y[:n, at:at + R + 64], pos, slots, cs, w, 1e-6, cache)
    no_error(dev)
    before = y.clone()
    for at in (R + 64, R + 64 + 192, R + 64 + H * 192 - 8):
        for n in (T, 1):
            with pytest.raises(RuntimeError, match="overlap kv"):
                ops.rope_latent_write(q[:n], y[:n, at:at + R + 64], pos, slots, cs, w, 1e-6, cache)
    assert torch.equal(y, before)
    no_error(dev)


# -------------------------------------------------------------------------- attention
class Cache:
    """Ragged contexts in permuted pages; what no sequence owns is NaN."""

    def __init__(self, dev, lens, R, page, seed, spare=2):
        g = torch.Generator(device=dev).manual_seed(seed)
        r = random.Random(seed)
        need = [-(-n // page) for n in lens]
        total = sum(need) + spare
        ids = list(range(total))
        r.shuffle(ids)
        self.cache = torch.full((total, page, R + 64), NAN, device=dev, dtype=torch.bfloat16)
        self.bt = torch.zeros(len(lens), max(need + [1]) + 1, dtype=torch.int32)
        self.rows, at = [], 0
        flat = self.cache.view(-1, R + 64)
        for i, n in enumerate(lens):
            self.bt[i, :need[i]] = torch.tensor(ids[at:at + need[i]], dtype=torch.int32)
            at += need[i]
            rows = torch.randn(n, R + 64, generator=g, device=dev).to(torch.bfloat16)
            j = torch.arange(n)
            flat[(self.bt[i, j // page].long() * page + j % page).to(dev)] = rows
            self.rows.append(rows)
        self.bt = self.bt.to(dev)
        self.ctx = torch.tensor(lens, dtype=torch.int32, device=dev)
        self.g = g

    def randn(self, *s, std=1.0):
        return (torch.randn(*s, generator=self.g, device=self.cache.device) * std).to(torch.bfloat16)


def decode64(q, rows, w, scale):
    """q [H, 192], rows [ctx, R + 64], w [H, 256, R] -> out [H, 128] and its standard deviation
    under the roundings of qa, p, o and out to bf16."""
    H, R = w.shape[0], w.shape[2]
    if rows.shape[0] == 0:
        z = torch.zeros(H, 128, dtype=torch.float64, device=q.device)
        return z, z
    q, rows, w = q.double(), rows.double(), w.double()
    c = rows[:, :R]
    qn = torch.einsum("hd,hdr->hr", q[:, :128], w[:, :128])
    s = (qn @ c.T + q[:, 128:] @ rows[:, R:].T) * scale
    p = torch.softmax(s, -1)
    o = p @ c
    out = torch.einsum("hr,hvr->hv", o, w[:, 128:])
    v = torch.einsum("kr,hvr->hkv", c, w[:, 128:])
    dev_v = p[..., None] * (v - out[:, None])  # d out / d s_j
    grad = torch.einsum("hkv,kr->hvr", dev_v, c) * scale  # d out / d qa_r
    var = torch.einsum("hvr,hr->hv", grad ** 2, qn ** 2)
    var += torch.einsum("hk,hkv->hv", p ** 2, v ** 2)
    var += torch.einsum("hr,hvr->hv", o ** 2, w[:, 128:] ** 2)
    var += out ** 2
    slop = F32 * torch.einsum("hk,hkv->hv", p, v.abs())
    return out, 8 * U / math.sqrt(3) * var.sqrt() + slop


def prefill64(q, rows, w, scale):
    """q [n, H, 192] at the end of rows [ctx, R + 64] -> out [n, H, 128] and its tolerance under the
    roundings of k, v, p and out to bf16."""
    n, H, _ = q.shape
    ctx, R = rows.shape[0], w.shape[2]
    q, rows, w = q.double(), rows.double(), w.double()
    out = torch.empty(n, H, 128, dtype=torch.float64, device=q.device)
    tol = torch.empty_like(out)
    seen = torch.arange(ctx, device=q.device)[None] <= torch.arange(ctx - n, ctx, device=q.device)[:, None]
    for h in range(H):
        kn, v = rows[:, :R] @ w[h, :128].T, rows[:, :R] @ w[h, 128:].T
        s = (q[:, h, :128] @ kn.T + q[:, h, 128:] @ rows[:, R:].T) * scale
        p = torch.softmax(s.masked_fill(~seen, -math.inf), -1)
        o = p @ v
        ds2 = (q[:, h, :128] ** 2 @ (kn ** 2).T) * scale ** 2  # variance of s_j in units of u^2 / 3
        a = p ** 2 * ds2
        var = a @ v ** 2 - 2 * o * (a @ v) + o ** 2 * a.sum(1, keepdim=True)
        var += 2 * (p ** 2 @ v ** 2) + o ** 2
        out[:, h] = o
        tol[:, h] = 8 * U / math.sqrt(3) * var.clamp_min(0).sqrt() + F32 * (p @ v.abs())
    return out, tol


LENS = [1, 15, 16, 17, 0, 63, 64, 65, 127, 128, 129, 300, 1000]


@pytest.mark.parametrize("H,R,page,max_ctx", [(1, 512, 16, None), (3, 256, 64, 1), (8, 512, 64, 100),
                                              (17, 512, 32, 1000), (28, 512, 16, 200), (64, 512, 16, None),
                                              (65, 256, 16, 0), (128, 512, 32, 1000), (33, 256, 32, 64),
                                              (200, 256, 16, None)])
def test_decode(dev, H, R, page, max_ctx):
    from kapsl_sdk_b200 import ops

    k = Cache(dev, LENS, R, page, H * 7 + R)
    B = len(LENS)
    qw = k.randn(B, H * 192 + 16, std=1.5)
    q = qw[:, 8:H * 192 + 8]  # a view of wider rows
    w = k.randn(H, 256, R, std=1 / math.sqrt(R))
    scale = 1 / math.sqrt(192)
    out = torch.full((B, H * 128 + 8), 3.0, device=dev, dtype=torch.bfloat16)
    ops.latent_decode_attention(q, k.cache, w, k.bt, k.ctx, H, out=out[:, :H * 128], max_ctx=max_ctx)
    no_error(dev)
    assert bool((out[:, H * 128:] == 3.0).all())
    for b in range(B):
        exp, tol = decode64(q[b].view(H, 192), k.rows[b], w, scale)
        within(out[b, :H * 128].view(H, 128), exp, tol)


@pytest.mark.parametrize("B,H,hi", [(40, 5, 700), (300, 3, 130), (2, 7, 20000), (17, 70, 900)])
def test_decode_ragged_batches(dev, B, H, hi):
    """Stretches of the schedule that hold many sequences, and sequences cut into many pieces;
    empty rows first, last and between."""
    from kapsl_sdk_b200 import ops

    r = random.Random(B)
    lens = [0 if r.random() < 0.15 else r.randint(1, hi) for _ in range(B)]
    if B > 2:
        lens[0] = lens[-1] = 0
    k = Cache(dev, lens, 512, 16, B + H)
    q, w = k.randn(B, H * 192, std=1.5), k.randn(H, 256, 512, std=1 / math.sqrt(512))
    out = ops.latent_decode_attention(q, k.cache, w, k.bt, k.ctx, H)
    no_error(dev)
    for b in sorted(r.sample(range(B), min(B, 24)) + [0, B - 1]):
        exp, tol = decode64(q[b].view(H, 192), k.rows[b], w, 1 / math.sqrt(192))
        within(out[b].view(H, 128), exp, tol)


def test_decode_large_logits(dev):
    """A running maximum that moves by far more than one tile's spread, in both directions."""
    from kapsl_sdk_b200 import ops

    H, R, lens = 9, 512, [700, 640, 129]
    k = Cache(dev, lens, R, 16, 5)
    q = k.randn(3, H * 192)
    w = k.randn(H, 256, R, std=1 / math.sqrt(R))
    flat = k.cache.view(-1, R + 64)
    for b, n in enumerate(lens):  # grow (b = 0), shrink (1) or spike (2) along the context
        f = torch.linspace(0.1, 6.0, n, device=dev) if b == 0 else torch.linspace(6.0, 0.1, n, device=dev)
        if b == 2:
            f = torch.full((n,), 0.2, device=dev)
            f[128] = 8.0
        rows = (k.rows[b].float() * f[:, None]).to(torch.bfloat16)
        j = torch.arange(n, device=dev)
        flat[k.bt[b, j // 16].long() * 16 + j % 16] = rows
        k.rows[b] = rows
    for max_ctx in (None, 64, 200):  # pieces of one tile, of many, whole sequences
        out = ops.latent_decode_attention(q, k.cache, w, k.bt, k.ctx, H, max_ctx=max_ctx)
        no_error(dev)
        for b in range(3):
            exp, tol = decode64(q[b].view(H, 192), k.rows[b], w, 1 / math.sqrt(192))
            within(out[b].view(H, 128), exp, tol)


@pytest.mark.parametrize("H,page,max_ctx", [(65, 16, None), (72, 32, 64), (128, 64, 300), (128, 16, 1000),
                                            (129, 16, None), (200, 32, 130), (257, 64, None)])
def test_decode_many_heads(dev, H, page, max_ctx):
    """CTA pairs: tiles of 128 keys whose second half is empty, begins or ends within; heads that fill
    no tile of 128, one, or several; no, one and many pieces a row."""
    from kapsl_sdk_b200 import ops

    lens = [128, 1, 0, 63, 64, 65, 127, 129, 191, 192, 193, 255, 256, 257, 900, 0]
    k = Cache(dev, lens, 512, page, H + page)
    qw, w = k.randn(len(lens), H * 192 + 8, std=1.5), k.randn(H, 256, 512, std=1 / math.sqrt(512))
    out = torch.full((len(lens) + 1, H * 128 + 8), 3.0, device=dev, dtype=torch.bfloat16)
    q = qw[:, :H * 192]
    ops.latent_decode_attention(q, k.cache, w, k.bt, k.ctx, H, out=out[:-1, :H * 128], max_ctx=max_ctx)
    no_error(dev)
    assert bool((out[:, H * 128:] == 3.0).all()) and bool((out[-1] == 3.0).all())
    for b in range(len(lens)):
        exp, tol = decode64(q[b].view(H, 192), k.rows[b], w, 1 / math.sqrt(192))
        within(out[b, :H * 128].view(H, 128), exp, tol)


def test_decode_many_heads_maxima_and_pages(dev):
    """Maxima that grow, shrink or jump along a context, in either CTA's keys; block table entries outside."""
    from kapsl_sdk_b200 import ops

    H, lens = 70, [700, 640, 330, 330]
    k = Cache(dev, lens, 512, 16, 8)
    q, w = k.randn(4, H * 192), k.randn(H, 256, 512, std=1 / math.sqrt(512))
    flat = k.cache.view(-1, 576)
    for b, n in enumerate(lens):
        f = torch.linspace(0.1, 6.0, n, device=dev) if b == 0 else torch.linspace(6.0, 0.1, n, device=dev)
        if b >= 2:
            f = torch.full((n,), 0.2, device=dev)
            f[140 if b == 2 else 200] = 8.0
        rows = (k.rows[b].float() * f[:, None]).to(torch.bfloat16)
        j = torch.arange(n, device=dev)
        flat[k.bt[b, j // 16].long() * 16 + j % 16] = rows
        k.rows[b] = rows
    for max_ctx in (None, 64, 256):
        good = ops.latent_decode_attention(q, k.cache, w, k.bt, k.ctx, H, max_ctx=max_ctx)
        no_error(dev)
        for b in range(4):
            exp, tol = decode64(q[b].view(H, 192), k.rows[b], w, 1 / math.sqrt(192))
            within(good[b].view(H, 128), exp, tol)
    for bad in (-1, k.cache.shape[0], 2 ** 31 - 1):
        bt = k.bt.clone()
        bt[1, 6] = bad
        out = ops.latent_decode_attention(q, k.cache, w, bt, k.ctx, H, max_ctx=256)
        torch.cuda.synchronize()
        assert ops.check_errors(dev) == 82
        assert torch.equal(out[[0, 2, 3]], good[[0, 2, 3]])


def test_decode_many_heads_graphs_and_streams(dev):
    """Captured, replayed and run on two streams at once: the eager results, bit for bit."""
    from kapsl_sdk_b200 import ops

    H = 128
    k = Cache(dev, [300, 77, 0, 1000] * 9, 512, 16, 10)
    w, q = k.randn(H * 256, 512, std=1 / math.sqrt(512)), k.randn(36, H * 192)

    def run():
        return ops.latent_decode_attention(q, k.cache, w, k.bt, k.ctx, H, max_ctx=1000)

    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = run()
    for _ in range(3):
        q.copy_(k.randn(36, H * 192))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(o, run())
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], []
    for _ in range(3):
        for st in streams:
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                got.append(run())
    torch.cuda.synchronize()
    assert all(torch.equal(g, o) for g in got)
    no_error(dev)


def test_prefill_absorbed_many_heads(dev):
    """New tokens one by one through the CTA pairs: neighbours in the batch share a block table."""
    from kapsl_sdk_b200 import ops

    q_lens, ctx_lens, H = [5, 1, 3], [300, 64, 3], 66
    k = Cache(dev, ctx_lens, 512, 32, 14)
    q, w = k.randn(9, H * 192, std=1.5), k.randn(H, 256, 512, std=1 / math.sqrt(512))
    plan = ops.latent_prefill_plan(q_lens, ctx_lens, dev)
    out = ops.latent_prefill_attention(q, k.cache, w, plan, k.bt, H, form="absorbed")
    no_error(dev)
    at = 0
    for s, (n, c) in enumerate(zip(q_lens, ctx_lens)):
        for i in range(n):
            exp, tol = decode64(q[at].view(H, 192), k.rows[s][:c - n + i + 1], w, 1 / math.sqrt(192))
            within(out[at].view(H, 128), exp, tol)
            at += 1


@pytest.mark.parametrize("form", ["single", "expanded", "absorbed"])
@pytest.mark.parametrize("H", [3, 66])
def test_first_keys_weigh_nothing(dev, form, H):
    """The first two tiles' scores are -inf (an infinite rotary value), the others far below zero: the
    result is the softmax over those."""
    from kapsl_sdk_b200 import ops

    ctx, n, scale = 400, 3, 1 / math.sqrt(192)
    k = Cache(dev, [ctx], 512, 16, 30)
    q, w = k.randn(n, H, 192), k.randn(H, 256, 512, std=1 / math.sqrt(512))
    q[..., 128] = 8.0
    rows = k.rows[0].clone()
    rows[:, 512] = -500.0
    j = torch.arange(ctx, device=dev)
    flat = k.cache.view(-1, 576)
    flat[k.bt[0, j // 16].long() * 16 + j % 16] = rows
    flat[k.bt[0, j[:256] // 16].long() * 16 + j[:256] % 16, 512] = -math.inf
    if form == "single":
        n = 1
        out = ops.latent_decode_attention(q[-1:].reshape(1, H * 192), k.cache, w, k.bt, k.ctx, H, max_ctx=64)
        q = q[-1:]
    else:
        plan = ops.latent_prefill_plan([n], [ctx], dev)
        out = ops.latent_prefill_attention(q.reshape(n, H * 192), k.cache, w, plan, k.bt, H, form=form)
    no_error(dev)
    for i in range(n):
        exp, tol = decode64(q[i], rows[256:ctx - n + i + 1], w, scale)
        kn = rows[256:ctx - n + i + 1, :512].double() @ w[:, :128].double().transpose(1, 2)  # keys, rounded to bf16
        vh = rows[256:ctx - n + i + 1, :512].double() @ w[:, 128:].double().transpose(1, 2)
        s = (torch.einsum("hd,hkd->hk", q[i, :, :128].double(), kn) +
             q[i, :, 128:].double() @ rows[256:ctx - n + i + 1, 512:].double().T) * scale
        p = torch.softmax(s, -1)
        ds2 = torch.einsum("hd,hkd->hk", q[i, :, :128].double() ** 2, kn ** 2) * scale ** 2
        var = torch.einsum("hk,hkv->hv", p ** 2 * ds2, (vh - exp[:, None]) ** 2)
        var += torch.einsum("hk,hkv->hv", p ** 2, vh ** 2)
        # scores of some -290: fp32 sums of 576 products err by 2^-24 * 24 * 290 in the exponent
        slop = 2.0 ** -24 * 24 * 290 * torch.einsum("hk,hkv->hv", p, vh.abs())
        within(out[i].view(H, 128), exp, tol + 8 * U / math.sqrt(3) * var.sqrt() + slop)


@pytest.mark.parametrize("H", [3, 66])
@pytest.mark.parametrize("n,first", [(3, 400), (200, 400), (400, 150)])
def test_rows_without_a_finite_score(dev, H, n, first):
    """The first keys' scores are -inf (an infinite rotary value).  A row that sees no others gives zeros in
    every form, with one key range or several, whatever its neighbours in the batch are."""
    from kapsl_sdk_b200 import ops

    lens, scale = [400, 30], 1 / math.sqrt(192)
    k = Cache(dev, lens, 512, 16, 31)
    q, w = k.randn(n + 5, H, 192), k.randn(H, 256, 512, std=1 / math.sqrt(512))
    q[:n, :, 128] = 8.0
    j = torch.arange(lens[0], device=dev)
    flat = k.cache.view(-1, 576)
    k.rows[0][:first, 512] = -math.inf
    flat[k.bt[0, j // 16].long() * 16 + j % 16] = k.rows[0]
    plan = ops.latent_prefill_plan([n, 5], lens, dev)
    outs = [ops.latent_prefill_attention(q.view(n + 5, -1), k.cache, w, plan, k.bt, H, form="expanded", key_ranges=r)
            for r in (1, 2, 4)]
    outs.append(ops.latent_prefill_attention(q.view(n + 5, -1), k.cache, w, plan, k.bt, H, form="absorbed"))
    empty = max(0, first - (lens[0] - n))  # rows that see the first keys only
    two = torch.stack([q[empty - 1], q[-1]]).view(2, -1)
    for max_ctx in (1, None):  # one piece, several
        ctx = torch.tensor([first, 30], dtype=torch.int32, device=dev)
        one = ops.latent_decode_attention(two, k.cache, w, k.bt, ctx, H, max_ctx=max_ctx)
        assert bool((one[0] == 0).all()) and bool(torch.isfinite(one[1].float()).all())
    no_error(dev)
    exp, tol = prefill64(q[n:], k.rows[1], w, scale)
    for i, out in enumerate(outs):
        assert bool((out[:empty] == 0).all())
        assert bool(torch.isfinite(out[empty:].float()).all())
        if i < 3:
            within(out[n:].view(5, H, 128), exp, tol)
            if empty < n:  # the others: softmax over the keys that count
                e, t = prefill64(q[empty:n], k.rows[0][first:], w, scale)
                within(out[empty:n].view(n - empty, H, 128), e, t)


def test_decode_pages_outside(dev):
    """A table entry outside the cache records an error; other rows are untouched by it."""
    from kapsl_sdk_b200 import ops

    k = Cache(dev, [40, 50], 512, 16, 3)
    q, w = k.randn(2, 5 * 192), k.randn(5, 256, 512, std=0.04)
    good = ops.latent_decode_attention(q, k.cache, w, k.bt, k.ctx, 5)
    no_error(dev)
    for bad in (-1, k.cache.shape[0], 2 ** 31 - 1):
        bt = k.bt.clone()
        bt[0, 1] = bad
        out = ops.latent_decode_attention(q, k.cache, w, bt, k.ctx, 5)
        torch.cuda.synchronize()
        assert ops.check_errors(dev) == 82
        assert torch.equal(out[1], good[1])
    # a context longer than its table is cut to the table
    ctx = torch.tensor([40, 10 ** 9], dtype=torch.int32, device=dev)
    out = ops.latent_decode_attention(q[1:], k.cache, w, k.bt[1:, :3].contiguous(), ctx[1:], 5, max_ctx=64)
    torch.cuda.synchronize()
    exp, tol = decode64(q[1].view(5, 192), k.rows[1][:48], w, 1 / math.sqrt(192))
    within(out[0].view(5, 128), exp, tol)
    no_error(dev)


def test_decode_refuses(dev):
    from kapsl_sdk_b200 import ops

    k = Cache(dev, [40, 50], 512, 16, 3)
    q, w = k.randn(2, 5 * 192), k.randn(5, 256, 512, std=0.04)
    a0 = dict(q=q, cache=k.cache, w=w, bt=k.bt, ctx=k.ctx, H=5, out=None)
    for kw in (dict(q=q.float()), dict(q=q[:, :-1]), dict(q=q.cpu()), dict(cache=k.cache[..., :448].contiguous()),
               dict(cache=k.cache.float()), dict(cache=k.cache[:, :8].contiguous()), dict(w=w[:4]), dict(H=4),
               dict(w=w[..., :256].contiguous()), dict(w=w.transpose(1, 2)), dict(bt=k.bt.long()), dict(bt=k.bt[:1]),
               dict(ctx=k.ctx.long()), dict(ctx=k.ctx[:1]), dict(out=q[:, :5 * 128]),
               dict(out=torch.empty(2, 5 * 128, device=dev)), dict(q=k.randn(2, 5 * 192 + 1)[:, 1:]), dict(H=0)):
        a = dict(a0)
        a.update(kw)
        with pytest.raises((RuntimeError, TypeError, ValueError)):
            ops.latent_decode_attention(a["q"], a["cache"], a["w"], a["bt"], a["ctx"], a["H"], out=a["out"])
    assert ops.latent_decode_attention(q[:0], k.cache, w, k.bt, k.ctx, 5).shape == (0, 640)
    no_error(dev)


@pytest.mark.parametrize("H", [3, 66, 300])
def test_one_row_of_any_pitch(dev, H):
    """A single row may be a view whose row stride no tensor map could take (dims of one index never step),
    and rows may share memory (an expanded query)."""
    from kapsl_sdk_b200 import ops

    k = Cache(dev, [70], 512, 16, 40)
    w, scale = k.randn(H, 256, 512, std=1 / math.sqrt(512)), 1 / math.sqrt(192)
    q = k.randn(1, H * 192 + 3)[:, :H * 192]
    assert q.stride(0) % 8 != 0
    plan = ops.latent_prefill_plan([1], [70], dev)
    exp, tol = decode64(q.view(H, 192), k.rows[0], w, scale)
    e2, t2 = prefill64(q.reshape(1, H, 192), k.rows[0], w, scale)
    for form, e, t in (("decode", exp, tol), ("absorbed", exp, tol), ("expanded", e2[0], t2[0])):
        out = torch.full((1, H * 128 + 3), 3.0, device=dev, dtype=torch.bfloat16)
        if form == "decode":
            ops.latent_decode_attention(q, k.cache, w, k.bt, k.ctx, H, out=out[:, :H * 128])
        else:
            ops.latent_prefill_attention(q, k.cache, w, plan, k.bt, H, out=out[:, :H * 128], form=form)
        no_error(dev)
        within(out[0, :H * 128].view(H, 128), e, t)
        assert bool((out[:, H * 128:] == 3.0).all())
    n = 5
    many = q[0].expand(n, H * 192)
    out = ops.latent_decode_attention(many, k.cache, w, k.bt.expand(n, -1).contiguous(), k.ctx.expand(n).contiguous(), H)
    within(out.view(n, H, 128), exp.expand(n, H, 128), tol.expand(n, H, 128))
    plan = ops.latent_prefill_plan([n], [70], dev)
    for form in ("absorbed", "expanded"):
        out = ops.latent_prefill_attention(many, k.cache, w, plan, k.bt, H, form=form)
        no_error(dev)
        e, t = (exp, tol) if form == "absorbed" else (e2[0], t2[0])
        within(out[-1].view(H, 128), e, t)


def test_decode_refuses_what_32_bits_do_not_count(dev):
    """Tables so wide, or rows so many, that tokens rounded up to a tile or the tiles of all rows pass 32 bits."""
    from kapsl_sdk_b200 import ops

    k = Cache(dev, [40], 512, 64, 3)
    w = k.randn(1, 256, 512, std=0.04)
    wide = torch.zeros(1, 2 ** 31 // 64 - 1, dtype=torch.int32, device=dev)
    with pytest.raises(RuntimeError, match="too wide"):
        ops.latent_decode_attention(k.randn(1, 192), k.cache, w, wide, k.ctx, 1)
    n, ctx = 65535, 2200000
    plan = ops.latent_prefill_plan([n], [ctx], dev)
    with pytest.raises(RuntimeError, match="too many"):
        ops.latent_prefill_attention(k.randn(n, 192), k.cache, w, plan, wide[:, :ctx // 64 + 1].contiguous(), 1,
                                     form="absorbed")
    # a wide table by itself is in order: entries behind the context are not looked at
    q = k.randn(1, 192)
    far = wide[:, :2 ** 24].contiguous()
    far[:, 2:] = -1
    far[:, :2] = k.bt[:, :1].expand(1, 2)
    exp, tol = decode64(q.view(1, 192), k.rows[0], w, 1 / math.sqrt(192))
    within(ops.latent_decode_attention(q, k.cache, w, far, k.ctx, 1).view(1, 128), exp, tol)
    no_error(dev)


PREFILLS = [([1], [1]), ([17], [17]), ([130], [130]), ([128, 256], [128, 300]), ([300, 0, 1, 64], [557, 9, 900, 64]),
            ([257, 129, 5, 385], [257, 513, 1000, 400]), ([128, 3, 100, 1, 64], [128, 129, 640, 2500, 385])]


@pytest.mark.parametrize("q_lens,ctx_lens", PREFILLS)
@pytest.mark.parametrize("form", ["expanded", "absorbed"])
@pytest.mark.parametrize("H,R,page", [(1, 512, 16), (5, 256, 64), (28, 512, 32)])
def test_prefill(dev, form, q_lens, ctx_lens, H, R, page):
    from kapsl_sdk_b200 import ops

    k = Cache(dev, ctx_lens, R, page, H + len(q_lens))
    T, q0 = sum(q_lens) + 5, 3  # rows before and behind the sequences
    qw = k.randn(T, H * 192 + 8, std=1.5)
    q = qw[:, :H * 192]
    w = k.randn(H * 256, R, std=1 / math.sqrt(R))
    out = torch.full((T, H * 128 + 8), 3.0, device=dev, dtype=torch.bfloat16)
    bt = torch.cat([k.bt.new_full((2, k.bt.shape[1]), -1), k.bt])
    plan = ops.latent_prefill_plan(q_lens, ctx_lens, dev, q_start=q0, bt_start=2)
    ops.latent_prefill_attention(q, k.cache, w, plan, bt, H, out=out[:, :H * 128], form=form)
    no_error(dev)
    at = q0
    for i, n in enumerate(q_lens):
        if n and form == "absorbed":  # a few tokens of each sequence, the ends among them
            for t in sorted({0, n - 1, n // 2, n // 3}):
                exp, tol = decode64(q[at + t].view(H, 192), k.rows[i][:ctx_lens[i] - n + t + 1], w.view(H, 256, R),
                                    1 / math.sqrt(192))
                within(out[at + t, :H * 128].view(H, 128), exp, tol)
        elif n:
            exp, tol = prefill64(q[at:at + n].view(n, H, 192), k.rows[i], w.view(H, 256, R), 1 / math.sqrt(192))
            within(out[at:at + n, :H * 128].view(n, H, 128), exp, tol)
        at += n
    assert bool((out[:q0] == 3.0).all()) and bool((out[at:] == 3.0).all()) and bool((out[:, H * 128:] == 3.0).all())


def test_prefill_passes_over_heads(dev, monkeypatch):
    """A small bound on the expanded rows cuts the heads into passes, the last one shorter."""
    from kapsl_sdk_b200 import ops

    k = Cache(dev, [200, 90], 512, 16, 11)
    H = 7
    q, w = k.randn(200, H * 192), k.randn(H * 256, 512, std=0.05)
    plan = ops.latent_prefill_plan([110, 90], [200, 90], dev)
    one = ops.latent_prefill_attention(q, k.cache, w, plan, k.bt, H, form="expanded")
    monkeypatch.setattr(ops, "LATENT_KV_BYTES", plan.kv_rows * 512 * 3)
    assert torch.equal(one, ops.latent_prefill_attention(q, k.cache, w, plan, k.bt, H, form="expanded"))
    no_error(dev)


@pytest.mark.parametrize("n", [20, 200])
def test_prefill_numbers_of_key_tiles(dev, n):
    """One to eleven key tiles, in the order of two row tiles and in that of one (the ring's barriers turn
    over at every second tile)."""
    from kapsl_sdk_b200 import ops

    H, R = 3, 512
    lens = [c for c in range(100, 1401, 65) if c >= n]
    k = Cache(dev, lens, R, 16, n)
    q, w = k.randn(n * len(lens), H * 192, std=1.5), k.randn(H * 256, R, std=1 / math.sqrt(R))
    plan = ops.latent_prefill_plan([n] * len(lens), lens, dev)
    out = ops.latent_prefill_attention(q, k.cache, w, plan, k.bt, H, form="expanded", key_ranges=1)
    no_error(dev)
    for i in range(len(lens)):
        exp, tol = prefill64(q[i * n:(i + 1) * n].view(n, H, 192), k.rows[i], w.view(H, 256, R), 1 / math.sqrt(192))
        within(out[i * n:(i + 1) * n].view(n, H, 128), exp, tol)


@pytest.mark.parametrize("key_ranges", [2, 3, 7, 32])
def test_prefill_key_ranges(dev, key_ranges):
    """The keys in parts: parts that end inside a row's keys, that only later rows see, that hold nothing."""
    from kapsl_sdk_b200 import ops

    q_lens, ctx_lens, H, R = [300, 20, 129, 1], [1100, 2000, 129, 7], 3, 512
    k = Cache(dev, ctx_lens, R, 16, 21)
    q, w = k.randn(sum(q_lens), H * 192, std=1.5), k.randn(H * 256, R, std=1 / math.sqrt(R))
    plan = ops.latent_prefill_plan(q_lens, ctx_lens, dev)
    out = ops.latent_prefill_attention(q, k.cache, w, plan, k.bt, H, form="expanded", key_ranges=key_ranges)
    no_error(dev)
    at = 0
    for i, n in enumerate(q_lens):
        exp, tol = prefill64(q[at:at + n].view(n, H, 192), k.rows[i], w.view(H, 256, R), 1 / math.sqrt(192))
        within(out[at:at + n].view(n, H, 128), exp, tol)
        at += n
    with pytest.raises(RuntimeError):
        ops.latent_prefill_attention(q, k.cache, w, plan, k.bt, H, form="expanded", key_ranges=33)


@pytest.mark.parametrize("key_ranges", [0, 2, 9])
def test_prefill_ranges_and_passes(dev, key_ranges, monkeypatch):
    """A long context cut into parts beside whole short ones, with the heads in several passes; rows between
    and behind the sequences stay."""
    from kapsl_sdk_b200 import ops

    q_lens, ctx_lens, H, R = [140, 3, 257, 1, 30], [6000, 3, 3100, 129, 700], 5, 512
    k = Cache(dev, ctx_lens, R, 16, 50)
    T, q0 = sum(q_lens) + 4, 2
    q, w = k.randn(T, H * 192, std=1.5), k.randn(H * 256, R, std=1 / math.sqrt(R))
    plan = ops.latent_prefill_plan(q_lens, ctx_lens, dev, q_start=q0)
    step, cut, part, slots = plan.passes(H, key_ranges)
    assert step == H and 0 < cut < plan.work.shape[0] and slots > 1
    outs = []
    for room in (ops.LATENT_KV_BYTES, 2 * (plan.kv_rows * 512 + cut * slots * ops.LATENT_PART_BYTES)):
        monkeypatch.setattr(ops, "LATENT_KV_BYTES", room)
        if outs:
            assert plan.passes(H, key_ranges or slots)[0] == 2  # heads 2, 2, 1
        out = torch.full((T, H * 128), 3.0, device=dev, dtype=torch.bfloat16)
        ops.latent_prefill_attention(q, k.cache, w, plan, k.bt, H, out=out, form="expanded",
                                     key_ranges=key_ranges or slots)
        outs.append(out)
    no_error(dev)
    assert torch.equal(*outs)
    at = q0
    for i, n in enumerate(q_lens):
        exp, tol = prefill64(q[at:at + n].view(n, H, 192), k.rows[i], w.view(H, 256, R), 1 / math.sqrt(192))
        within(out[at:at + n].view(n, H, 128), exp, tol)
        at += n
    assert bool((out[:q0] == 3.0).all()) and bool((out[at:] == 3.0).all())


def test_prefill_picks_a_form(dev):
    """Few tokens over a long context go by themselves, a long chunk is expanded; the result is that of the
    form named."""
    from kapsl_sdk_b200 import ops

    for q_lens, ctx_lens, H, form in (([3, 1], [900, 300], 8, "absorbed"), ([600], [700], 30, "expanded")):
        k = Cache(dev, ctx_lens, 512, 16, 2)
        q, w = k.randn(sum(q_lens), H * 192), k.randn(H * 256, 512, std=0.05)
        plan = ops.latent_prefill_plan(q_lens, ctx_lens, dev)
        assert plan.absorbed_is_shorter(H) == (form == "absorbed")
        assert torch.equal(ops.latent_prefill_attention(q, k.cache, w, plan, k.bt, H),
                           ops.latent_prefill_attention(q, k.cache, w, plan, k.bt, H, form=form))
    with pytest.raises(ValueError):
        ops.latent_prefill_attention(q, k.cache, w, plan, k.bt, H, form="folded")
    no_error(dev)


def test_prefill_large_logits(dev):
    from kapsl_sdk_b200 import ops

    H, R, n = 2, 512, 520
    k = Cache(dev, [n], R, 16, 6)
    f = torch.linspace(0.1, 5.0, n, device=dev)
    f[300:] = f[300:].flip(0)
    rows = (k.rows[0].float() * f[:, None]).to(torch.bfloat16)
    j = torch.arange(n, device=dev)
    k.cache.view(-1, R + 64)[k.bt[0, j // 16].long() * 16 + j % 16] = rows
    q, w = k.randn(n, H * 192), k.randn(H * 256, R, std=1 / math.sqrt(R))
    out = ops.latent_prefill_attention(q, k.cache, w, ops.latent_prefill_plan([n], [n], dev), k.bt, H, form="expanded")
    no_error(dev)
    exp, tol = prefill64(q.view(n, H, 192), rows, w.view(H, 256, R), 1 / math.sqrt(192))
    within(out.view(n, H, 128), exp, tol)


def far_scores(dev, n, H, ctx, mag, kind, R=512):
    """Scores of mag times small numbers, exact in fp32 (a product of two short rotary values): the largest
    are equal, all others far below, so the result is the mean over the equal ones, however
    large mag is.  Every other query prefers the smallest rotary values."""
    k = Cache(dev, [ctx], R, 16, n + ctx)
    q, w = torch.zeros(n, H, 192, device=dev, dtype=torch.bfloat16), k.randn(H * 256, R, std=1 / math.sqrt(R))
    q[:, :, 128] = 2.0 ** (mag // 2)
    q[::2, :, 128] *= -1
    j = torch.arange(ctx, device=dev)
    f = {"mixed": 0.5 + j * 7 % 5, "growing": 1.0 + j // 100, "above zero": 4.0 + j * 3 % 2}[kind]
    rows = k.rows[0]
    rows[:, R:] = 0
    rows[:, R] = f * 2.0 ** (mag - mag // 2) * (1 if kind == "above zero" else -1)
    k.cache.view(-1, R + 64)[k.bt[0, j // 16].long() * 16 + j % 16] = rows
    return k, q, w, rows


@pytest.mark.parametrize("kind", ["mixed", "growing", "above zero"])
@pytest.mark.parametrize("mag", [20, 26, 31, 36, 60, 110])
@pytest.mark.parametrize("n,ctx", [(3, 700), (300, 700)])
def test_prefill_far_scores(dev, n, ctx, mag, kind):
    """Scores whose last place in fp32 is worth more than the steps in which the running maximum is raised."""
    from kapsl_sdk_b200 import ops

    H = 2
    k, q, w, rows = far_scores(dev, n, H, ctx, mag, kind)
    plan = ops.latent_prefill_plan([n], [ctx], dev)
    out = ops.latent_prefill_attention(q.view(n, -1), k.cache, w, plan, k.bt, H, form="expanded", key_ranges=1)
    no_error(dev)
    exp, tol = prefill64(q, rows, w.view(H, 256, 512), 1 / math.sqrt(192))
    within(out.view(n, H, 128), exp, tol)


@pytest.mark.parametrize("kind", ["mixed", "growing", "above zero"])
@pytest.mark.parametrize("mag", [20, 26, 31, 36, 60, 110])
@pytest.mark.parametrize("H", [2, 66])
def test_decode_far_scores(dev, H, mag, kind):
    """The same for single tokens, each context one piece."""
    from kapsl_sdk_b200 import ops

    k, q, w, rows = far_scores(dev, 2, H, 700, mag, kind)
    for i in range(2):
        out = ops.latent_decode_attention(q[i:i + 1].view(1, -1), k.cache, w, k.bt, k.ctx, H, max_ctx=1)
        no_error(dev)
        exp, tol = decode64(q[i], rows, w.view(H, 256, 512), 1 / math.sqrt(192))
        within(out.view(H, 128), exp, tol)


@pytest.mark.parametrize("kind", ["mixed", "growing", "above zero"])
@pytest.mark.parametrize("mag", [20, 26, 36, 110])
@pytest.mark.parametrize("H", [2, 66])
def test_pieces_of_far_scores(dev, H, mag, kind):
    """Equal largest scores in several pieces of a context count one by one, not piece by piece."""
    from kapsl_sdk_b200 import ops

    n, ctx, scale = 4, 700, 1 / math.sqrt(192)
    k, q, w, rows = far_scores(dev, n, H, ctx, mag, kind)
    plan = ops.latent_prefill_plan([n], [ctx], dev)
    flat = q.view(n, -1)
    got = [ops.latent_prefill_attention(flat, k.cache, w, plan, k.bt, H, form="expanded", key_ranges=r) for r in (2, 5)]
    exp, tol = prefill64(q, rows, w.view(H, 256, 512), scale)
    one = ops.latent_decode_attention(flat[-1:], k.cache, w, k.bt, k.ctx, H)
    rows_alone = ops.latent_prefill_attention(flat, k.cache, w, plan, k.bt, H, form="absorbed")
    no_error(dev)
    for out in got:
        within(out.view(n, H, 128), exp, tol)
    for i in range(n):
        exp, tol = decode64(q[i], rows[:ctx - n + i + 1], w.view(H, 256, 512), scale)
        within(rows_alone[i].view(H, 128), exp, tol)
    within(one.view(H, 128), exp, tol)


@pytest.mark.parametrize("form", ["expanded", "absorbed"])
def test_prefill_pages_outside_and_refusals(dev, form):
    from kapsl_sdk_b200 import ops

    k = Cache(dev, [40, 50], 512, 16, 3)
    q, w = k.randn(50, 5 * 192), k.randn(5, 256, 512, std=0.04)
    plan = ops.latent_prefill_plan([20, 30], [40, 50], dev)
    good = ops.latent_prefill_attention(q, k.cache, w, plan, k.bt, 5, form=form)
    no_error(dev)
    for bad in (-1, k.cache.shape[0], 2 ** 31 - 1):
        bt = k.bt.clone()
        bt[0, 1] = bad
        out = ops.latent_prefill_attention(q, k.cache, w, plan, bt, 5, form=form)
        torch.cuda.synchronize()
        assert ops.check_errors(dev) == 82
        assert torch.equal(out[20:], good[20:]) and torch.isfinite(out.float()).all()
    wide = ops.latent_prefill_plan([20, 30], [40, 5000], dev)
    for bad in (lambda: ops.latent_prefill_attention(q[:49], k.cache, w, plan, k.bt, 5),
                lambda: ops.latent_prefill_attention(q, k.cache, w, plan, k.bt[:1], 5),
                lambda: ops.latent_prefill_attention(q, k.cache, w, wide, k.bt, 5),
                lambda: ops.latent_prefill_attention(q, k.cache, w, plan, k.bt, 4),
                lambda: ops.latent_prefill_attention(q.float(), k.cache, w, plan, k.bt, 5),
                lambda: ops.latent_prefill_attention(q, k.cache.float(), w, plan, k.bt, 5),
                lambda: ops.latent_prefill_attention(q, k.cache, w[:4], plan, k.bt, 5),
                lambda: ops.latent_prefill_attention(q, k.cache, w, plan, k.bt, 5, out=q[:, :640])):
        with pytest.raises((RuntimeError, TypeError)):
            bad()
    empty = ops.latent_prefill_plan([0], [0], dev)
    assert bool((ops.latent_prefill_attention(q, k.cache, w, empty, k.bt, 5) == 0).all())
    no_error(dev)


@pytest.mark.parametrize("scale", [0.0, -0.05, 1.0])
def test_scales(dev, scale):
    """Scale 0 weighs every key alike, a negative one prefers the least similar, a large one a single key."""
    from kapsl_sdk_b200 import ops

    H, R, n, ctx = 3, 512, 70, 200
    k = Cache(dev, [ctx], R, 16, 12)
    q, w = k.randn(n, H * 192), k.randn(H * 256, R, std=1 / math.sqrt(R))
    plan = ops.latent_prefill_plan([n], [ctx], dev)
    out = ops.latent_prefill_attention(q, k.cache, w, plan, k.bt, H, scale=scale, form="expanded")
    exp, tol = prefill64(q.view(n, H, 192), k.rows[0], w.view(H, 256, R), scale)
    within(out.view(n, H, 128), exp, tol)
    one = ops.latent_decode_attention(q[-1:], k.cache, w, k.bt, k.ctx, H, scale=scale)
    exp, tol = decode64(q[-1].view(H, 192), k.rows[0], w.view(H, 256, R), scale)
    within(one.view(H, 128), exp, tol)
    no_error(dev)


def test_cache_past_32_bit_offsets(dev):
    """Pages whose elements lie more than 2^31 from the cache's start: write, decode, both prefill forms."""
    from kapsl_sdk_b200 import ops
    from kapsl_sdk_b200.ops import reference as ref

    page, R, H, n = 64, 512, 4, 150
    blocks = 2 ** 31 // (page * (R + 64)) + 40
    cache = torch.empty(blocks, page, R + 64, dtype=torch.bfloat16, device=dev)
    g = torch.Generator(device=dev).manual_seed(8)

    def rn(*s, std=1.0):
        return (torch.randn(*s, generator=g, device=dev) * std).to(torch.bfloat16)

    bt = torch.tensor([[blocks - 1, 3, blocks - 7]], dtype=torch.int32, device=dev)
    pos = torch.arange(n, device=dev, dtype=torch.int32)
    slots = bt[0].long()[pos.long() // page] * page + pos.long() % page
    cs = ref.rope_cos_sin(n, 64, 1e4, device=dev)
    kv, q, wn, w = rn(n, R + 64), rn(n, H, 192), 1 + rn(R, std=0.1), rn(H * 256, R, std=1 / math.sqrt(R))
    ops.rope_latent_write(q[..., 128:], kv, pos, slots, cs, wn, 1e-5, cache)
    rows = cache.view(-1, R + 64)[slots]
    exp = ref.latent_row(kv, pos, cs, wn, 1e-5)
    assert float((rows.float() - exp).abs().max()) < 2 * U * float(exp.abs().max())
    plan = ops.latent_prefill_plan([40], [n], dev)
    q2 = q[-40:].reshape(40, -1)
    got = ops.latent_prefill_attention(q2, cache, w, plan, bt, H, form="expanded")
    e, t = prefill64(q[-40:], rows, w.view(H, 256, R), 1 / math.sqrt(192))
    within(got.view(40, H, 128), e, t)
    got = ops.latent_prefill_attention(q2, cache, w, plan, bt, H, form="absorbed")
    one = ops.latent_decode_attention(q2[-1:], cache, w, bt, torch.tensor([n], dtype=torch.int32, device=dev), H)
    e, t = decode64(q[-1], rows, w.view(H, 256, R), 1 / math.sqrt(192))
    within(got[-1].view(H, 128), e, t)
    within(one[0].view(H, 128), e, t)
    no_error(dev)


def test_write_from_one_projection(dev):
    """Queries and latents as views of one projection's rows, rotated in place: its other columns stay."""
    from kapsl_sdk_b200 import ops
    from kapsl_sdk_b200.ops import reference as ref

    T, H, R = 9, 3, 256
    g = torch.Generator(device=dev).manual_seed(2)
    y = torch.randn(T, H * 192 + R + 64, generator=g, device=dev).to(torch.bfloat16)
    before = y.clone()
    q, kv = y[:, :H * 192].view(T, H, 192), y[:, H * 192:]
    cs = ref.rope_cos_sin(50, 64, 1e4, device=dev)
    pos = torch.randint(0, 50, (T,), generator=g, device=dev, dtype=torch.int32)
    cache = torch.zeros(1, 16, R + 64, dtype=torch.bfloat16, device=dev)
    w = torch.ones(R, dtype=torch.bfloat16, device=dev)
    ops.rope_latent_write(q[..., 128:], kv, pos, torch.arange(T, device=dev), cs, w, 1e-6, cache, interleaved=True)
    exp, mag = rope64(before[:, :H * 192].view(T, H, 192)[..., 128:], pos, cs, 0, True)
    within(q[..., 128:], exp, U * exp.abs() + 2.0 ** -22 * mag)
    assert torch.equal(q[..., :128], before[:, :H * 192].view(T, H, 192)[..., :128])
    assert torch.equal(kv, before[:, H * 192:])
    c = before[:, H * 192:H * 192 + R].double()
    lat = c / (c.pow(2).mean(1, keepdim=True) + 1e-6).sqrt()
    within(cache[0, :T, :R], lat, lat.abs() * (U + 2.0 ** -18))
    no_error(dev)


def test_graphs_streams_and_repeats(dev):
    """Two captured graphs replayed in turn and eager calls on two streams give the eager results."""
    from kapsl_sdk_b200 import ops

    H, R = 20, 512
    k = Cache(dev, [300, 77, 0, 1000], R, 16, 9)
    w = k.randn(H * 256, R, std=1 / math.sqrt(R))
    qd, qp = k.randn(4, H * 192), k.randn(177, H * 192)
    plan = ops.latent_prefill_plan([100, 77], [300, 77], dev)

    def decode():
        return ops.latent_decode_attention(qd, k.cache, w, k.bt, k.ctx, H, max_ctx=1000)

    def prefill():
        return ops.latent_prefill_attention(qp, k.cache, w, plan, k.bt, H, form="expanded")

    decode(), prefill()
    torch.cuda.synchronize()
    graphs = []
    for fn in (decode, prefill):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            o = fn()
        graphs.append((gr, o, fn))
    for rep in range(3):
        qd.copy_(k.randn(4, H * 192))
        qp.copy_(k.randn(177, H * 192))
        exp = [fn().clone() for _, _, fn in graphs]
        for gr, _, _ in graphs:
            gr.replay()
        torch.cuda.synchronize()
        for (_, o, _), e in zip(graphs, exp):
            assert torch.equal(o, e)
    s = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for rep in range(4):
        for i, fn in enumerate((decode, prefill)):
            s[i].wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s[i]):
                got[i].append(fn())
    torch.cuda.synchronize()
    for i in range(2):
        for o in got[i]:
            assert torch.equal(o, exp[i])
    no_error(dev)


@pytest.mark.parametrize("H,R", [(20, 512), (128, 512), (70, 256)])
def test_captured_decode_follows_lengths_and_tables(dev, H, R):
    """A captured call replayed with other lengths and block tables: longer and shorter contexts, rows that
    became empty or filled, the eager results bit for bit."""
    from kapsl_sdk_b200 import ops

    k = Cache(dev, [900, 33, 400, 1, 700, 64], R, 16, H)
    B = len(k.rows)
    q, w = k.randn(B, H * 192), k.randn(H * 256, R, std=1 / math.sqrt(R))
    bt, ctx = k.bt.clone(), torch.tensor([10, 0, 400, 1, 0, 64], dtype=torch.int32, device=dev)

    def run():
        return ops.latent_decode_attention(q, k.cache, w, bt, ctx, H)

    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for order, lens in (((0, 1, 2, 3, 4, 5), (900, 33, 400, 1, 700, 64)), ((4, 2, 0, 5, 3, 1), (650, 0, 899, 17, 1, 33)),
                        ((5, 4, 3, 2, 1, 0), (0, 0, 0, 0, 0, 0)), ((2, 2, 2, 2, 2, 2), (400, 128, 129, 1, 0, 16))):
        bt.copy_(k.bt[list(order)])
        ctx.copy_(torch.tensor(lens, dtype=torch.int32))
        q.copy_(k.randn(B, H * 192))
        for _ in range(2):
            graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        assert torch.equal(got, run())
        for b in range(B):
            exp, tol = decode64(q[b].view(H, 192), k.rows[order[b]][:lens[b]], w.view(H, 256, R), 1 / math.sqrt(192))
            within(got[b].view(H, 128), exp, tol)
    no_error(dev)


def test_captured_prefill_in_parts(dev):
    """A captured call whose long context is cut, replayed with other queries and beside eager calls on another
    stream."""
    from kapsl_sdk_b200 import ops

    H, q_lens, ctx_lens = 4, [200, 30], [5000, 300]
    k = Cache(dev, ctx_lens, 512, 16, 60)
    q, w = k.randn(230, H * 192), k.randn(H * 256, 512, std=1 / math.sqrt(512))
    plan = ops.latent_prefill_plan(q_lens, ctx_lens, dev)
    assert plan.passes(H)[1] == 1 and plan.work.shape[0] == 2

    def run():
        return ops.latent_prefill_attention(q, k.cache, w, plan, k.bt, H, form="expanded")

    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    side = torch.cuda.Stream()
    for _ in range(3):
        q.copy_(k.randn(230, H * 192))
        exp = run()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = [run() for _ in range(3)]
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, exp) and all(torch.equal(o, exp) for o in other)
    no_error(dev)


def test_layer_run_together(dev):
    """A latent-attention layer as a serving loop drives it: two prefill chunks of one sequence
    beside a whole prompt of another, then decode steps of both, against a 64-bit layer that
    sees the full sequences.  The cache holds bf16 rows, which the oracle rounds likewise."""
    from kapsl_sdk_b200 import ops
    from kapsl_sdk_b200.ops import reference as ref

    g = torch.Generator(device=dev).manual_seed(4)
    H, R, page, lens = 5, 256, 16, [90, 41]

    def rn(*s, std=1.0):
        return (torch.randn(*s, generator=g, device=dev) * std).to(torch.bfloat16)

    w, wn = rn(H * 256, R, std=1 / math.sqrt(R)), 1 + rn(R, std=0.1)
    cs = ref.rope_cos_sin(200, 64, 1e4, device=dev)
    Q = [rn(n, H * 192, std=1.5) for n in lens]
    KV = [rn(n, R + 64) for n in lens]
    cache = torch.full((14, page, R + 64), NAN, device=dev, dtype=torch.bfloat16)
    bt = torch.randperm(14, generator=g, device=dev).int()[:12].view(2, 6).contiguous()
    scale = 0.06
    outs = [[], []]
    done = [0, 0]

    def step(news, prefill):
        rows = [(s, done[s] + i) for s, n in enumerate(news) for i in range(n)]
        q = torch.cat([Q[s][done[s]:done[s] + n] for s, n in enumerate(news)]).clone()
        kv = torch.cat([KV[s][done[s]:done[s] + n] for s, n in enumerate(news)])
        pos = torch.tensor([p for _, p in rows], dtype=torch.int32, device=dev)
        slots = torch.tensor([int(bt[s, p // page]) * page + p % page for s, p in rows], device=dev)
        ops.rope_latent_write(q.view(-1, H, 192)[..., 128:], kv, pos, slots, cs, wn, 1e-5, cache, interleaved=True)
        for s, n in enumerate(news):
            done[s] += n
        if prefill:
            plan = ops.latent_prefill_plan(news, done, dev)
            o = ops.latent_prefill_attention(q, cache, w, plan, bt, H, scale=scale, form="expanded")
        else:
            ctx = torch.tensor(done, dtype=torch.int32, device=dev)
            o = ops.latent_decode_attention(q, cache, w, bt, ctx, H, scale=scale, max_ctx=max(done))
        for s, n in enumerate(news):
            outs[s].append(o[:n])
            o = o[n:]

    step([50, 0], True)
    step([30, 31], True)
    for _ in range(10):
        step([1, 1], False)
    no_error(dev)
    for s, n in enumerate(lens):
        pos = torch.arange(n, device=dev)
        rows = ref.latent_row(KV[s], pos, cs, wn, 1e-5, interleaved=True).to(torch.bfloat16)
        q = ref.rope(Q[s].view(n, H, 192), pos, cs, offset=128, interleaved=True).to(torch.bfloat16)
        got = torch.cat(outs[s]).view(n, H, 128)
        exp, tol = prefill64(q, rows, w.view(H, 256, R), scale)
        first = n - 10
        within(got[:first], exp[:first], tol[:first])
        for i in range(first, n):
            e, t = decode64(q[i], rows[:i + 1], w.view(H, 256, R), scale)
            within(got[i], e, t)
