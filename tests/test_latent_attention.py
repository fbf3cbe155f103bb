"""Latent attention's plans and plain forms on the CPU (no GPU needed)."""
import math

import pytest
import torch

from kapsl_sdk_b200 import ops
from kapsl_sdk_b200.ops import reference as ref


def test_plan_rows_and_tiles():
    p = ops.latent_prefill_plan([300, 0, 1, 17], [557, 40, 900, 17], device="cpu", q_start=5, bt_start=2)
    # contexts start at multiples of 16; a sequence without new tokens needs no context
    assert p.seq_info.tolist() == [[5, 300, 557, 2, 0], [305, 0, 0, 3, 560], [305, 1, 900, 4, 560],
                                   [306, 17, 17, 5, 1472]]
    assert (p.rows, p.tables, p.max_ctx, p.kv_rows) == (323, 6, 900, 1504)
    # every query row in exactly one tile, most keys first
    got = [(s, t) for s, t in p.work.tolist()]
    assert got == [(2, 0), (0, 256), (0, 0), (3, 0)]
    # every 128 context rows once
    assert p.kv_work.tolist() == [[0, r] for r in range(0, 557, 128)] + [[2, r] for r in range(0, 900, 128)] + [[3, 0]]
    # every new token by itself
    assert p.row_ctx.tolist() == list(range(258, 558)) + [900] + list(range(1, 18))
    assert p.row_table.tolist() == [2] * 300 + [4] + [5] * 17
    assert p.single_tiles == sum(-(-c // 64) for c in p.row_ctx.tolist())


def test_plan_key_ranges():
    def ranges(q_lens, ctx_lens, heads):
        return ops.latent_prefill_plan(q_lens, ctx_lens, device="cpu").key_ranges(heads)

    assert ranges([512], [16384], 20) == 3      # few row tiles over a long context
    assert ranges([20], [4020], 8) == 8         # never under 4 key tiles a part
    assert ranges([2048] * 4, [8192] * 4, 128) == 1  # a full GPU
    assert ranges([17, 1], [17, 300], 4) == 1   # short contexts
    assert ranges([256], [200000], 1) == 32     # what the join takes


def test_plan_of_nothing():
    p = ops.latent_prefill_plan([], [], device="cpu")
    assert p.work.shape == (0, 2) and p.seq_info.shape == (0, 5) and p.kv_rows == 0 and p.tables == 0
    p = ops.latent_prefill_plan([0, 0], [0, 7], device="cpu")
    assert p.work.shape == (0, 2) and p.kv_rows == 0


@pytest.mark.parametrize("q_lens,ctx_lens", [([5], [4]), ([-1], [4]), ([1, 2], [3])])
def test_plan_refuses(q_lens, ctx_lens):
    with pytest.raises(ValueError):
        ops.latent_prefill_plan(q_lens, ctx_lens, device="cpu")
    with pytest.raises(ValueError):
        ops.latent_prefill_plan([1], [1], device="cpu", q_start=-1)


def test_reference_rope_layouts():
    # the interleaved layout is the half layout of permuted dims
    g = torch.Generator().manual_seed(0)
    x = torch.randn(9, 3, 80, generator=g)
    pos = torch.randint(0, 50, (9,), generator=g)
    cs = ref.rope_cos_sin(50, 32, 10000.0)
    il = ref.rope(x, pos, cs, offset=16, interleaved=True)
    assert torch.equal(il[..., :16], x[..., :16]) and torch.equal(il[..., 48:], x[..., 48:])
    perm = torch.cat([torch.arange(0, 32, 2), torch.arange(1, 32, 2)])
    half = ref.rope(x[..., 16:48][..., perm], pos, cs)
    assert torch.equal(il[..., 16:48][..., perm], half)
    # against the complex product, in 64 bits
    z = torch.view_as_complex(x[..., 16:48].double().reshape(9, 3, 16, 2))
    c = cs[pos].double()
    y = torch.view_as_real(z * torch.complex(c[:, None, :16], c[:, None, 16:])).reshape(9, 3, 32)
    assert (il[..., 16:48] - y).abs().max() < 4 * 2.0 ** -24 * 8


def test_reference_forms_agree():
    """The absorbed order of the products gives the expanded form's result."""
    g = torch.Generator().manual_seed(1)
    H, R, ctx, n = 3, 256, 37, 5
    q = torch.randn(n, H, 192, generator=g).double()
    rows = torch.randn(ctx, R + 64, generator=g).double()
    w = (torch.randn(H, 256, R, generator=g) / math.sqrt(R)).double()
    got = ref.latent_attention(q, rows, w.reshape(-1, R), 0.07)
    for i in range(n):
        c = rows[:ctx - n + i + 1]
        qa = torch.cat([torch.einsum("hd,hdr->hr", q[i, :, :128], w[:, :128]), q[i, :, 128:]], -1)
        o = torch.softmax(qa @ c.T * 0.07, -1) @ c[:, :R]
        exp = torch.einsum("hr,hvr->hv", o, w[:, 128:])
        assert (got[i].double() - exp).abs().max() < 1e-4


def test_reference_rows_without_a_finite_score():
    g = torch.Generator().manual_seed(3)
    H, R, ctx, n = 2, 256, 9, 7
    q, rows = torch.randn(n, H, 192, generator=g), torch.randn(ctx, R + 64, generator=g)
    w = torch.randn(H * 256, R, generator=g) / math.sqrt(R)
    q[..., 128] = 1.0
    rows[:5, R] = -math.inf  # new tokens 0 - 2 see keys up to 2 - 4
    out = ref.latent_attention(q, rows, w, 0.07)
    assert bool((out[:3] == 0).all()) and bool(torch.isfinite(out).all())
    rest = ref.latent_attention(q[3:], rows[5:], w, 0.07)
    # the same keys with weights of 0 between them: sums of at most 9 values
    assert (out[3:] - rest).abs().max() <= 16 * 2.0 ** -24 * rest.abs().max() * 9


@pytest.mark.parametrize("q_lens,ctx_lens,heads", [
    ([256] + [1] * 500, [65536] + [64] * 500, 8), ([512] + [17] * 1000, [30000] + [40] * 1000, 4),
    ([256] + [40] * 1000, [131072] + [40] * 1000, 8), ([256] + [80] * 100, [65536] + [80] * 100, 16)])
def test_partial_results_of_mixed_batches(q_lens, ctx_lens, heads):
    """Short sequences beside a long context are not cut with it, and need no partial results."""
    p = ops.latent_prefill_plan(q_lens, ctx_lens, device="cpu")
    step, cut, part, slots = p.passes(heads)
    assert step == heads and cut == -(-q_lens[0] // 256) and part >= 4 and slots == p.key_ranges(heads) > 1
    assert cut * slots * step * ops.LATENT_PART_BYTES < 80 << 20
    # every tile in order, the parts cover the longest
    assert p.key_tiles == sorted(p.key_tiles, reverse=True) and len(p.key_tiles) == p.work.shape[0]
    assert slots * part >= p.key_tiles[0] and all(n <= part for n in p.key_tiles[cut:])


@pytest.mark.parametrize("q_lens,ctx_lens,heads,ranges", [
    ([4096] * 8, [20000] * 8, 128, 32), ([256] * 900, [2000] * 900, 16, 32), ([300] * 40, [9000] * 40, 20, 7),
    ([64], [500], 5, 32), ([2048] * 300, [3000] * 300, 2, 32)])
def test_scratch_of_prefill_is_bounded(q_lens, ctx_lens, heads, ranges):
    """However many parts are asked for, what a pass holds stays within the bound while one head's keys and
    values do."""
    p = ops.latent_prefill_plan(q_lens, ctx_lens, device="cpu")
    step, cut, part, slots = p.passes(heads, ranges)
    assert 1 <= step <= heads and slots <= 32
    room = cut * slots * ops.LATENT_PART_BYTES
    assert room <= ops.LATENT_KV_BYTES
    assert step == 1 or step * (p.kv_rows * 512 + room) <= ops.LATENT_KV_BYTES
    assert p.passes(heads, 1)[1:] == (0, 0, 1)


def test_check_errors_of_a_device_without_kernels():
    """Asking for the CPU's status is answered, and keeps no buffer of it as a GPU's."""
    before = dict(ops._err_bufs)
    assert ops.check_errors(torch.device("cpu")) == 0
    assert ops._err_bufs == before
    with pytest.raises(RuntimeError):
        ops.error_buffer(torch.device("cpu"))


def test_passes_of_nothing():
    p = ops.latent_prefill_plan([0], [0], device="cpu")
    assert p.passes(7) == p.passes(7, 4) == (7, 0, 0, 1)
