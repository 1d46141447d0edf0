"""The 8-bit paged cache and its operators against plain 64-bit forms, through the Python
entry points (C ABI).

Bounds, derived from the arithmetic and fixed before the first run:

* rotary: three f32 roundings and one to the output type;
* append, read, fork, compact: bit for bit (IEEE division, round-half-even, moved bytes);
* attend: the output's own rounding (half an ulp), the softmax weights' rounding to 16 bits
  (2^-11 of sum p|v|) and f32 sums and exponentials (2^-13 of sum p|v| covers logits up to
  about 500 in f32 with margin);
* lse: f32 logits, 2e-5 of max(1, |lse|).
"""
from __future__ import annotations

import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

HALF_ULP = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8, "f32": 2.0 ** -24}  # finfo.eps / 2


def types():
    import torch
    return {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def ints(v, cuda):
    import torch
    return torch.tensor(v, dtype=torch.int32, device=cuda)


def row_starts(new):
    return [0, *np.cumsum(new).tolist()]


def rope_table(positions, rot, cuda, interleaved=False):
    from ffn_residual_mesh_b200.kvcache import RotaryTable
    return RotaryTable(rot, positions, interleaved=interleaved, device=cuda)


def make_tables(lengths, P, rng, spare=3, width=None):
    """Pages of each sequence in a random order of a pool with a few spare ones."""
    counts = [-(-n // P) for n in lengths]
    pages = sum(counts) + spare
    order, at, rows = rng.permutation(pages).tolist(), 0, []
    width = max(counts + [1]) + 1 if width is None else width
    for n in counts:
        rows.append(order[at:at + n] + [-1] * (width - n))
        at += n
    return rows, pages, order[at:]


def make_cache(cuda, pages, H, D, P, layers=1, max_seqs=64, seed=0, dead=()):
    """A filled cache; pages in `dead` have NaN scales and the lowest code everywhere."""
    import torch
    from ffn_residual_mesh_b200.kvcache import PagedKvCache
    g = torch.Generator(device=cuda).manual_seed(seed)
    cache = PagedKvCache(layers, pages, H, D, page_tokens=P, max_seqs=max_seqs)
    for codes, scale in ((cache.k_codes, cache.k_scale), (cache.v_codes, cache.v_scale)):
        codes.copy_((torch.randn(codes.shape, device=cuda, generator=g) * 40).round().clamp(-127, 127))
        scale.copy_(0.01 + 0.04 * torch.rand(scale.shape, device=cuda, generator=g))
        for page in dead:
            scale[:, page] = math.nan
            codes[:, page] = -128
    return cache


# ---------------------------------------------------------------------------------- rotary
@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("dim,rot", [(128, 128), (128, 64), (96, 96), (80, 40), (64, 2), (66, 36), (256, 256)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary(cuda, dtype, dim, rot, interleaved):
    import torch
    import kv_reference as ref
    from ffn_residual_mesh_b200.kvcache import rotary
    table = rope_table(500, rot, cuda, interleaved)
    for T, heads in ((1, 1), (7, 5), (130, 3)):
        g = torch.Generator(device=cuda).manual_seed(T)
        x = torch.randn(T, heads + 2, dim, device=cuda, generator=g).to(types()[dtype])[:, 1:heads + 1]  # strided
        pos = torch.randint(0, 500, (T,), device=cuda, generator=g, dtype=torch.int32)
        for inverse in (False, True):
            y = rotary(x, pos, table, inverse=inverse)
            want = ref.rotate(x, table.cos_sin, pos.long(), interleaved, inverse)
            # |a||c| + |b||s| of a channel's pair, whose products and sum are rounded
            pair = torch.maximum(*(ref.rotate(x.abs(), table.cos_sin.abs(), pos.long(), interleaved, way)
                                   for way in (False, True)))
            bound = HALF_ULP[dtype] * want.abs() + 3 * 2.0 ** -24 * pair.abs() + 1e-7
            assert ((y.double() - want).abs() <= bound).all()
            assert torch.equal(y[..., rot:], x[..., rot:])
        # in place, and back again
        z = x.clone()
        rotary(z, pos, table, out=z)
        assert torch.equal(z, rotary(x, pos, table))
        rotary(z, pos, table, out=z, inverse=True)
        assert (z.double() - x.double()).abs().max() <= 4 * HALF_ULP[dtype] * 2 * x.abs().max().item() + 1e-6


def test_rotary_unaligned_rows_and_positions_outside(cuda):
    import torch
    import kv_reference as ref
    from ffn_residual_mesh_b200.kvcache import rotary
    table = rope_table(50, 64, cuda)
    flat = torch.randn(1 + 9 * 3 * 67, device=cuda).half()
    x = flat[1:].view(9, 3, 67)[..., :64]  # odd base and strides
    pos = ints([0, 49, 50, -1, 3, 2 ** 31 - 1, 1, 1, 0], cuda)
    y = rotary(x, pos, table)
    good = torch.tensor([0, 1, 4, 6, 7, 8], device=cuda)
    want = ref.rotate(x[good], table.cos_sin, pos[good].long())
    assert ((y[good].double() - want).abs() <= 2.0 ** -11 * want.abs() + 2e-6).all()
    assert torch.isnan(y[[2, 3, 5]]).all()


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_inverse_is_the_gradient(cuda, interleaved):
    """d sum(w * rotary(x)) / dx = inverse rotation of w: against the formula (the transposed
    matrix, built channel by channel in 64 bits) and against differences."""
    import torch
    import kv_reference as ref
    from ffn_residual_mesh_b200.kvcache import rotary
    table = rope_table(40, 32, cuda, interleaved)
    pos = ints([0, 7, 39], cuda)
    g = torch.Generator(device=cuda).manual_seed(1)
    w = torch.randn(3, 2, 48, device=cuda, generator=g)
    got = rotary(w, pos, table, inverse=True)
    eye = torch.eye(48, device=cuda, dtype=torch.float64)
    for t in range(3):
        matrix = ref.rotate(eye[:, None], table.cos_sin, pos[t].long().repeat(48), interleaved)[:, 0]  # row i: image of e_i
        want = w[t].double() @ matrix.T
        assert ((got[t].double() - want).abs() <= 1e-6 * (1 + want.abs())).all()
    x = torch.randn(3, 2, 48, device=cuda, generator=g)
    for d in (0, 1, 15, 16, 31, 32, 47):
        step = torch.zeros_like(x)
        step[..., d] = 2.0 ** -6
        diff = (rotary(x + step, pos, table).double() - rotary(x - step, pos, table).double()) / 2.0 ** -5
        # linear in x: only f32 rounding of values up to ~5 over the step is left
        assert (((diff * w.double()).sum(-1) - got[..., d].double()).abs() <= 48 * 2.0 ** -23 * 5 * 32 * 3).all()


# ---------------------------------------------------------------------------------- append, read
def check_append(cuda, new, held, H, D, P, dtype, group=0, rot=0, interleaved=False, seed=0, spread=1.0, x_of=None,
                 with_starts=True, strided=True):
    import torch
    import kv_reference as ref
    rng = np.random.default_rng(seed)
    lengths = [a + b for a, b in zip(new, held)]
    rows, pages, dead = make_tables(lengths, P, rng)
    cache = make_cache(cuda, pages, H, D, P, layers=2, seed=seed, dead=dead)
    cache.k_scale.mul_(0.3)  # most blocks grow, some do not
    starts = row_starts(new)
    T = starts[-1]
    g = torch.Generator(device=cuda).manual_seed(seed + 1)
    qkv = torch.randn(T, (group + 2) * H, D, device=cuda, generator=g) * spread
    if x_of is not None:
        x_of(qkv)
    qkv = qkv.to(types()[dtype])
    q, k, v = qkv[:, :group * H], qkv[:, group * H:(group + 1) * H], qkv[:, (group + 1) * H:]
    if not strided:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    table = rope_table(max(lengths) + 1, rot, cuda, interleaved) if rot else None
    before = [t.clone() for t in (cache.k_codes, cache.k_scale, cache.v_codes, cache.v_scale)]
    tables, lens = ints(rows, cuda), ints(lengths, cuda)
    st = ints(starts, cuda) if with_starts else None
    q_out = cache.append(1, k, v, tables, lens, starts=st, rope=table, q=q if group else None)
    cache.check()
    pos = torch.cat([torch.arange(a, a + b) for a, b in zip(held, new)]).to(cuda)
    kf = ref.rotate_f32(k, table.cos_sin, pos, interleaved) if rot else k.float()
    want = [t.cpu() for t in before]
    ref.append(want[0][1], want[1][1], kf.cpu(), rows, lengths, starts)
    ref.append(want[2][1], want[3][1], v.float().cpu(), rows, lengths, starts)
    for got, exp in zip((cache.k_codes, cache.k_scale, cache.v_codes, cache.v_scale), want):
        assert torch.equal(torch.nan_to_num(got.cpu().float(), -1.0), torch.nan_to_num(exp.float(), -1.0))
    if group:
        want_q = ref.rotate(q, table.cos_sin, pos, interleaved)
        assert ((q_out.double() - want_q).abs() <= HALF_ULP[dtype] * want_q.abs() + 2e-6 * spread).all()
    # read: code * scale of the same rows
    for kind, dt in types().items():
        rk, rv = cache.read(1, tables, lens, ints(starts, cuda), T, dtype=dt)
        cache.check()
        for got, codes, scale in ((rk, want[0][1], want[1][1]), (rv, want[2][1], want[3][1])):
            exp = torch.stack([codes[rows[b][p // P], :, p % P].float() * scale[rows[b][p // P]][:, None]
                               for b, (a, n) in enumerate(zip(held, new)) for p in range(a, a + n)])
            assert torch.equal(torch.nan_to_num(got.cpu(), -1.0), torch.nan_to_num(exp.to(dt), -1.0))
    return cache


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("H,D,P,rot,interleaved", [(2, 64, 16, 64, False), (1, 128, 64, 64, True), (3, 128, 32, 36, False),
                                                   (2, 256, 128, 256, False), (5, 64, 128, 0, False), (1, 256, 16, 10, True)])
def test_append(cuda, dtype, H, D, P, rot, interleaved):
    new, held = [1, P, 3 * P + 5, 2, P - 1, 1], [0, P, 7, P - 1, 1, 2 * P]
    check_append(cuda, new, held, H, D, P, dtype, group=3 if rot else 0, rot=rot, interleaved=interleaved, seed=H + D)


@pytest.mark.parametrize("strided", [True, False])
def test_append_single_tokens(cuda, strided):
    held = [0, 1, 15, 16, 17, 63, 64, 200, 31, 32]
    check_append(cuda, [1] * len(held), held, 8, 128, 16, "f16", group=8, rot=128, seed=3, with_starts=False, strided=strided)


def test_append_no_new_tokens_and_zero_values(cuda):
    def zeros(x):
        x[3:6] = 0
        x[:, -1] = 0
    check_append(cuda, [3, 0, 4, 0, 1], [5, 9, 0, 0, 3], 2, 64, 16, "bf16", seed=5, x_of=zeros)


def test_append_non_finite_values_mark_their_block(cuda):
    import torch
    def odd(x):
        x[0, 0, 3] = math.nan
        x[1, 1, 0] = math.inf
        x[20, 2, 5] = -math.inf
    cache = check_append(cuda, [17, 5], [3, 30], 2, 64, 16, "f32", seed=6, x_of=odd)
    assert torch.isnan(cache.k_scale[1]).any() and torch.isnan(cache.v_scale[1]).any()


@pytest.mark.parametrize("scale", [1.0, 3e-9, 1e-14, 7e-38, 1e30, 3e38 / 9])
def test_append_quotients_of_every_size(cuda, scale):
    """Values from the smallest to the largest: the codes are the IEEE quotients' still."""
    check_append(cuda, [64, 40], [0, 9], 2, 64, 32, "f32", seed=11, spread=scale)
    if scale in (1.0, 1e30):
        check_append(cuda, [300, 200], [5, 0], 4, 128, 64, "bf16", seed=12, spread=scale)  # ties


def test_append_token_by_token_stays_near_the_values(cuda):
    """200 single appends: a code's error is at most half a step at its own write and half a
    step of the then larger scale at each growth; with growths of a fixed ratio 1.05 or more
    the sum stays below 1/2 + 1/2 * sum 1.05^-i <= 11 steps of the last scale, and is in fact
    far below: 2 steps are asked for the mean, 11 for the largest."""
    import torch
    H, D, P = 2, 64, 64
    cache = make_cache(cuda, 8, H, D, P)
    g = torch.Generator(device=cuda).manual_seed(9)
    x = torch.randn(200, H, D, device=cuda, generator=g)
    tables = ints([[3, 1, 7, 0, -1]], cuda)
    for t in range(200):
        cache.append(0, x[t:t + 1], x[t:t + 1], tables, ints([t + 1], cuda))
    k, v = cache.read(0, tables, ints([200], cuda), ints([0, 200], cuda), 200)
    cache.check()
    page = torch.tensor([3, 1, 7, 0], device=cuda)[torch.arange(200, device=cuda) // P]
    step = cache.k_scale[0][page][..., None]
    assert torch.equal(k, v)
    assert ((k - x).abs() / step).max() <= 11 and ((k - x).abs() / step).mean() <= 2


def test_append_idle_and_impossible_sequences(cuda):
    import torch
    cache = make_cache(cuda, 6, 1, 64, 16)
    before = [t.clone() for t in (cache.k_codes, cache.k_scale)]
    x = torch.randn(4, 1, 64, device=cuda).half()
    table = rope_table(8, 64, cuda)
    q = cache.append(0, x, x, ints([[0, 1], [2, 3], [4, 5], [-1, -1]], cuda), ints([0, 3, 0, 0], cuda), rope=table, q=x)
    cache.check()
    assert (q[[0, 2, 3]] == 0).all() and torch.equal(cache.k_codes[0, :2], before[0][0, :2])

    def refused(error, tables, lengths, starts=None, rope=None):
        held = [t.clone() for t in (cache.k_codes, cache.k_scale, cache.v_codes, cache.v_scale)]
        rows = x[:starts[-1]] if starts else x[:len(lengths)]
        cache.append(0, rows, rows, ints(tables, cuda), ints(lengths, cuda), starts=ints(starts, cuda) if starts else None,
                     rope=rope)
        with pytest.raises(error):
            cache.check()
        cache.check()  # reported once
        for a, b in zip(held, (cache.k_codes, cache.k_scale, cache.v_codes, cache.v_scale)):
            assert torch.equal(a, b)

    refused(RuntimeError, [[6, 0]], [1])           # page past the pool
    refused(RuntimeError, [[-1, 0]], [5])          # no page
    refused(RuntimeError, [[0, 1]], [33])          # more than the table addresses
    refused(RuntimeError, [[0, 1]], [-2])
    refused(RuntimeError, [[0, 1]], [2], [0, 3])   # more new tokens than tokens
    refused(RuntimeError, [[0, 1]], [9], rope=table)  # position 8 of an 8-row table


# ---------------------------------------------------------------------------------- attend
def check_attend(cuda, new, lengths, H, G, D, P, dtype="f16", seed=0, causal=True, window=0, scale=None, spread=1.0,
                 with_starts=True, strided=False, spare=3, tamper=None, layers=1):
    import torch
    import kv_reference as ref
    rng = np.random.default_rng(seed)
    rows, pages, dead = make_tables(lengths, P, rng, spare)
    cache = make_cache(cuda, pages, H, D, P, layers=layers, seed=seed, dead=dead, max_seqs=max(64, len(lengths)))
    starts = row_starts(new)
    T = starts[-1]
    g = torch.Generator(device=cuda).manual_seed(seed + 5)
    pad = 2 if strided else 0
    q = (torch.randn(T, H * G + pad, D, device=cuda, generator=g) * spread).to(types()[dtype])[:, pad:]
    if tamper:
        tamper(cache, rows, q)
    out = torch.full((T + 1, H * G + pad, D), 7.0, device=cuda, dtype=types()[dtype])
    lse = torch.full((T, H * G), 7.0, device=cuda)
    L = layers - 1
    cache.attend(L, q, ints(rows, cuda), ints(lengths, cuda), starts=ints(starts, cuda) if with_starts else None,
                 out=out[:T, pad:], lse=lse, causal=causal, window=window, scale=scale)
    cache.check()
    assert (out[T] == 7).all() and (out[:, :pad] == 7).all(), "wrote past its rows"
    want, mag, want_lse = ref.attend(q, cache.k_codes[L], cache.k_scale[L], cache.v_codes[L], cache.v_scale[L], rows, lengths,
                                     starts, scale, causal, window)
    got = out[:T, pad:].double()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    fine = ~torch.isnan(want)
    bound = HALF_ULP[dtype] * want.abs() + (2.0 ** -11 + 2.0 ** -13) * mag + 1e-6
    excess = ((got - want).abs() - bound)[fine]
    assert excess.numel() == 0 or excess.max() <= 0, f"excess {excess.max().item():.3e}"
    empty = want_lse == -math.inf
    assert torch.equal(lse == -math.inf, empty) and (got[empty] == 0).all()
    ok = ~empty & ~torch.isnan(want_lse) & ~torch.isnan(want).any(-1)  # a row that sees a NaN scale is NaN, its lse too
    assert ((lse.double() - want_lse).abs()[ok] <= 2e-5 * want_lse.abs().clamp(min=1)[ok]).all()
    # the same bits again
    again = torch.empty_like(out[:T, pad:])
    cache.attend(L, q, ints(rows, cuda), ints(lengths, cuda), starts=ints(starts, cuda) if with_starts else None, out=again,
                 causal=causal, window=window, scale=scale)
    assert torch.equal(torch.nan_to_num(again, 9.0), torch.nan_to_num(out[:T, pad:], 9.0)), "not the same bits twice"
    return cache


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("P", [16, 32, 64, 128])
def test_attend_single_tokens(cuda, dtype, D, P):
    lengths = [1, 2, 15, 16, 17, 0, 63, 64, 65, 127, 128, 129, 1000, 333]
    for H, G in ((2, 4), (1, 8)):
        check_attend(cuda, [1] * len(lengths), lengths, H, G, D, P, dtype, seed=D + P + G, with_starts=False)


@pytest.mark.parametrize("n", [31, 32, 33, 64, 65, 200, 500])
def test_attend_many_sequences(cuda, n):
    """Batches over several runs of 32 sequences, idle slots and rowless ones among them."""
    rng = np.random.default_rng(n)
    lengths = rng.integers(0, 80, n).tolist()
    lengths[n // 2] = 1500
    check_attend(cuda, [1] * n, lengths, 2, 4, 64, 16, seed=n, with_starts=False)
    new = [min(int(k), x) for k, x in zip(rng.integers(0, 6, n), lengths)]
    check_attend(cuda, new, lengths, 1, 3, 128, 32, "bf16", seed=n)


@pytest.mark.parametrize("H,G", [(1, 1), (8, 1), (2, 3), (1, 7), (3, 5), (1, 16), (2, 12), (1, 33), (1, 64)])
def test_attend_head_groups(cuda, H, G):
    check_attend(cuda, [1] * 5, [700, 1, 0, 64, 129], H, G, 128, 64, seed=G, with_starts=False, strided=True)


@pytest.mark.parametrize("D,P", [(64, 16), (128, 64), (128, 128), (256, 32)])
@pytest.mark.parametrize("new,lengths", [
    ([5, 0, 1, 8, 3], [5, 9, 400, 8, 131]),          # a few tokens each, one sequence without rows
    ([300, 1, 129, 64], [300, 2000, 700, 64]),       # prompt chunks beside single tokens
    ([1], [257]), ([257], [257]), ([256], [256]), ([31, 33], [31, 1057])])
def test_attend_several_tokens(cuda, D, P, new, lengths):
    for H, G, dtype in ((2, 4, "f16"), (1, 5, "bf16")):
        check_attend(cuda, new, lengths, H, G, D, P, dtype, seed=len(new) + D, strided=G == 5)


@pytest.mark.parametrize("window", [1, 7, 16, 100, 128, 5000, 2 ** 31 - 1])
def test_attend_window(cuda, window):
    check_attend(cuda, [1] * 4, [1, 90, 1500, 128], 2, 4, 128, 16, seed=window, window=window, with_starts=False)
    check_attend(cuda, [200, 3, 128], [333, 500, 128], 2, 4, 128, 32, seed=window, window=window)


def test_attend_window_with_pages_given_back(cuda):
    """Pages that lie wholly before the window may be gone from the table."""
    def drop(cache, rows, q):
        rows[0][:10] = [-1] * 10
        rows[1][:3] = [99999] * 3
    check_attend(cuda, [1, 1], [300, 200], 2, 4, 128, 16, seed=2, window=100, with_starts=False, tamper=drop)
    check_attend(cuda, [20, 70], [300, 220], 2, 4, 128, 16, seed=3, window=100, tamper=drop)


def test_attend_all_keys(cuda):
    check_attend(cuda, [4, 150, 1], [100, 150, 700], 2, 4, 128, 64, seed=1, causal=False)
    check_attend(cuda, [4, 150], [100, 333], 2, 4, 64, 32, seed=1, causal=False, window=50)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_attend_large_logits_and_scales(cuda, dtype):
    """Logits of several hundred (one key takes all the weight), and queries past f16's range."""
    check_attend(cuda, [1, 40], [600, 300], 2, 4, 128, 64, dtype, seed=4, spread=20.0)
    check_attend(cuda, [1, 40], [600, 300], 2, 4, 128, 64, dtype, seed=4, scale=1e-3)
    if dtype == "bf16":
        check_attend(cuda, [1, 40], [600, 300], 2, 4, 128, 64, dtype, seed=4, spread=1e6, scale=1e-7)


def test_attend_scales_of_every_size(cuda):
    """Pages of zeros (the smallest scale), tiny and large value scales side by side."""
    def uneven(cache, rows, q):
        for i, s in enumerate((1e-12, 1e-6, 50.0, 1.0)):
            cache.v_scale[0, rows[0][i]] = s
            cache.v_scale[0, rows[1][i]] = s
        cache.v_codes[0, rows[0][0]] = 0
        cache.k_scale[0, rows[0][1]] = 1e-12
    check_attend(cuda, [1, 60], [300, 300], 2, 4, 128, 32, seed=8, tamper=uneven)
    check_attend(cuda, [1, 1], [300, 300], 2, 4, 128, 32, seed=8, tamper=uneven, with_starts=False)


def test_attend_nan_blocks_reach_the_rows_that_see_them(cuda):
    def poison(cache, rows, q):
        cache.k_scale[0, rows[0][2], 0] = math.nan   # tokens 32..47 of sequence 0, kv head 0
        cache.v_scale[0, rows[1][1], 1] = math.nan
    check_attend(cuda, [1, 1], [100, 100], 2, 4, 64, 16, seed=8, tamper=poison, with_starts=False)
    check_attend(cuda, [100, 100], [100, 100], 2, 4, 64, 16, seed=8, tamper=poison)
    check_attend(cuda, [1, 60], [100, 100], 2, 4, 64, 16, seed=8, tamper=poison, window=30)


def test_attend_nan_query_stays_in_its_row(cuda):
    import torch
    cache = make_cache(cuda, 8, 2, 128, 64)
    tables = ints([[0, 1, 2, 3], [4, 5, 6, 7]], cuda)
    for new in ([1, 1], [150, 100]):
        T = sum(new)
        q = torch.randn(T, 8, 128, device=cuda).half()
        args = dict(starts=ints(row_starts(new), cuda))
        base = cache.attend(0, q, tables, ints([200, 256], cuda), **args)
        q[0, 3, 5] = math.nan
        got = cache.attend(0, q, tables, ints([200, 256], cuda), **args)
        assert torch.isnan(got[0, 3]).all()
        got[0, 3] = base[0, 3]
        assert torch.equal(got, base)


def test_attend_rows_of_no_sequence_are_zero(cuda):
    import torch
    cache = make_cache(cuda, 8, 2, 128, 64)
    q = torch.randn(9, 8, 128, device=cuda).half()
    out = cache.attend(0, q, ints([[0, 1], [2, 3]], cuda), ints([100, 70], cuda), starts=ints([0, 3, 5], cuda))
    cache.check()
    assert (out[5:] == 0).all() and (out[:5] != 0).any(-1).all()


def test_attend_long_context(cuda):
    check_attend(cuda, [1, 1], [70001, 33], 1, 8, 128, 64, seed=1, with_starts=False)
    check_attend(cuda, [130], [20000], 1, 4, 128, 128, seed=1)


def test_attend_pool_past_32_bit_offsets(cuda):
    """Codes of one layer beyond 2^31 bytes: pages at the far end, written and read."""
    import torch
    import kv_reference as ref
    from ffn_residual_mesh_b200.kvcache import PagedKvCache
    pages, H, D, P = 18000, 8, 128, 128  # 2.36e9 codes
    cache = PagedKvCache(1, pages, H, D, page_tokens=P, max_seqs=4)
    rows = [[pages - 1, 5, pages - 3, -1], [pages - 2, 17000, -1, -1]]
    T = 300 + 140
    g = torch.Generator(device=cuda).manual_seed(3)
    k, v = (torch.randn(T, H, D, device=cuda, generator=g).half() for _ in range(2))
    tables, lengths, starts = ints(rows, cuda), ints([300, 140], cuda), ints([0, 300, 440], cuda)
    cache.append(0, k, v, tables, lengths, starts=starts)
    rk, _ = cache.read(0, tables, lengths, starts, T)
    assert (rk - k.float()).abs().max() <= 0.51 * cache.k_scale.max()
    for new in ([300, 140], [1, 1]):
        q = torch.randn(sum(new), H * 4, D, device=cuda, generator=g).half()
        out = cache.attend(0, q, tables, lengths, starts=ints(row_starts(new), cuda))
        cache.check()
        want, mag, _ = ref.attend(q, cache.k_codes[0], cache.k_scale[0], cache.v_codes[0], cache.v_scale[0], rows, [300, 140],
                                  row_starts(new))
        assert ((out.double() - want).abs() <= 2.0 ** -11 * want.abs() + (2.0 ** -11 + 2.0 ** -13) * mag + 1e-6).all()


def test_attend_unusable_data_is_recorded(cuda):
    import torch
    cache = make_cache(cuda, 4, 2, 64, 16)
    q = torch.randn(3, 4, 64, device=cuda).half()

    def refused(tables, lengths, starts=None):
        rows = starts[-1] if starts and 0 <= starts[-1] <= 3 else len(lengths)
        cache.attend(0, q[:rows], ints(tables, cuda), ints(lengths, cuda), starts=ints(starts, cuda) if starts else None)
        with pytest.raises(RuntimeError):
            cache.check()
        cache.check()

    refused([[4, 0]], [20])
    refused([[0, -1]], [20])
    refused([[0, 1]], [33])
    refused([[0, 1]], [-1])
    refused([[0, 1]], [2], [0, 3])
    out = cache.attend(0, q[:1], ints([[0, 1]], cuda), ints([20], cuda))  # and works on
    cache.check()
    assert torch.isfinite(out).all()


def test_attend_on_another_stream_and_in_a_graph(cuda):
    import torch
    from ffn_residual_mesh_b200.graphs import StepGraph
    cache = make_cache(cuda, 64, 2, 128, 16)
    rng = np.random.default_rng(0)
    rows, _, _ = make_tables([400, 33, 1], 16, rng, spare=0)
    rows = [[p % 64 for p in r] for r in rows]
    q = torch.randn(3, 16, 128, device=cuda).half()
    tables, lengths = ints(rows, cuda), ints([400, 33, 1], cuda)
    want = cache.attend(0, q, tables, lengths)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    out = torch.empty_like(q)
    cache.attend(0, q, tables, lengths, out=out, stream=side)
    side.synchronize()
    assert torch.equal(out, want)
    k = torch.randn(3, 2, 128, device=cuda).half()
    table = rope_table(512, 128, cuda)
    q_rot = torch.empty_like(q)

    def step():
        cache.append(0, k, k, tables, lengths, rope=table, q=q, q_out=q_rot)
        cache.attend(0, q_rot, tables, lengths, out=out)

    graph = StepGraph(step)
    lengths.copy_(ints([390, 30, 2], cuda))  # other lengths in place, the same graph
    graph.replay()
    torch.cuda.synchronize()
    got = out.clone()
    step()
    torch.cuda.synchronize()
    assert torch.equal(out, got)
    cache.check()
    graph.close()


# ---------------------------------------------------------------------------------- pages
@pytest.mark.parametrize("P,layers", [(16, 1), (64, 3), (128, 2)])
def test_fork(cuda, P, layers):
    import torch
    import kv_reference as ref
    lengths = [3 * P + 5, 1, P, 0, 2 * P - 1, P + 1]
    for seed, (parents, extra) in enumerate([
            ([0, 1, 2, 3, 4, 5], [1] * 6),                       # nobody forks
            ([0, 0, 0, 4, 4, -1, 2, 2], [1, 0, P, 3 * P, 1, 5, 1, 0]),
            ([5, -1, 5, 0, 1, 1, 1], [0, 0, 2, 7, 0, 1, 2]),
            ([-1, -1], [0, 2 * P + 1]),                          # everything freed
            ([4], [0]), ([3, 3], [0, 4])]):
        rng = np.random.default_rng(seed)
        rows, pages, _ = make_tables(lengths, P, rng, spare=17)
        cache = make_cache(cuda, pages, 2, 64, P, layers=layers, seed=seed)
        before = [t.clone() for t in (cache.k_codes, cache.k_scale, cache.v_codes, cache.v_scale)]
        width = 9
        out = torch.full((len(parents), width), 77, dtype=torch.int32, device=cuda)
        tables, lens, info = cache.fork(ints(rows, cuda), ints(lengths, cuda), ints(parents, cuda), ints(extra, cuda), out_tables=out)
        cache.check()
        want, want_len, copies = ref.fork(rows, lengths, parents, extra, pages, P, width)
        assert tables.tolist() == want and lens.tolist() == want_len
        held = {x for r in want for x in r if x >= 0}
        assert info.tolist() == [len(held), pages - len(held), len(copies), 0]
        for t, b in zip((cache.k_codes, cache.k_scale, cache.v_codes, cache.v_scale), before):
            for src, dst in copies:
                b[:, dst] = b[:, src]
            assert torch.equal(t, b)


def test_fork_after_a_rollback_into_a_shared_page(cuda):
    """A sequence cut back into a page that another still holds in full gets its own copy."""
    import kv_reference as ref
    cache = make_cache(cuda, 12, 1, 64, 16)
    rows, lengths = [[3, 5, -1], [3, 5, 7]], [20, 40]  # sequence 0 was cut from 32 or more
    tables, lens, info = cache.fork(ints(rows, cuda), ints(lengths, cuda), ints([0, 1], cuda), ints([1, 1], cuda))
    cache.check()
    assert tables.tolist() == ref.fork(rows, lengths, [0, 1], [1, 1], 12, 16, 3)[0]
    assert tables[0, 1] != 5 and tables[1].tolist() == [3, 5, 7] and info[2] == 1


def test_fork_short_of_pages_changes_nothing(cuda):
    import torch
    cache = make_cache(cuda, 5, 1, 64, 16)
    before = cache.k_codes.clone()
    args = ints([[0, 1, 2, -1]], cuda), ints([40], cuda)
    tables, lens, info = cache.fork(*args, ints([0, 0, 0, 0], cuda), ints([1] * 4, cuda))
    with pytest.raises(MemoryError):
        cache.check()
    assert (tables == -1).all() and (lens == 0).all() and info[2:].tolist() == [0, 1]
    assert torch.equal(cache.k_codes, before)
    tables, lens, info = cache.fork(*args, ints([0, 0, 0], cuda), ints([1] * 3, cuda))
    cache.check()
    assert info.tolist() == [5, 0, 2, 0]


def test_fork_unusable_tables(cuda):
    cache = make_cache(cuda, 5, 1, 64, 16)
    for rows, lengths, parents, extra in (([[0, 9]], [20], [0], [1]), ([[0, -1]], [20], [0], [1]), ([[0, 1]], [99], [0], [1]),
                                          ([[0, 1]], [20], [1], [1]), ([[0, 1]], [20], [-2], [1]), ([[0, 1]], [20], [0], [-1]),
                                          ([[0, 1]], [20], [0], [13]), ([[0, 1]], [20], [0], [2 ** 31 - 1])):
        tables, lens, info = cache.fork(ints(rows, cuda), ints(lengths, cuda), ints(parents, cuda), ints(extra, cuda))
        with pytest.raises(RuntimeError):
            cache.check()
        assert (tables == -1).all() and (lens == 0).all()


def test_fork_large_pool_and_batch(cuda):
    import torch
    import kv_reference as ref
    rng = np.random.default_rng(4)
    P, n = 16, 300
    lengths = rng.integers(0, 300, n).tolist()
    rows, pages, _ = make_tables(lengths, P, rng, spare=40000)
    cache = make_cache(cuda, pages, 1, 64, P, max_seqs=1500)
    parents = rng.integers(-1, n, 1500).tolist()
    extra = rng.integers(0, 40, 1500).tolist()
    width = 24
    out = torch.empty((1500, width), dtype=torch.int32, device=cuda)
    tables, lens, info = cache.fork(ints(rows, cuda), ints(lengths, cuda), ints(parents, cuda), ints(extra, cuda), out_tables=out)
    cache.check()
    want, want_len, copies = ref.fork(rows, lengths, parents, extra, pages, P, width)
    assert tables.tolist() == want and lens.tolist() == want_len and info[2] == len(copies)


@pytest.mark.parametrize("P,spare,n", [(16, 0, 5), (16, 40, 9), (64, 900, 30), (32, 70000, 200)])
def test_compact(cuda, P, spare, n):
    import torch
    import kv_reference as ref
    rng = np.random.default_rng(spare)
    lengths = rng.integers(0, 20 * P, n).tolist()
    lengths[0] = 0
    rows, pages, _ = make_tables(lengths, P, rng, spare)
    rows.append(rows[1])  # shared pages
    lengths.append(lengths[1])
    layers = 2 if pages < 5000 else 1
    cache = make_cache(cuda, pages, 1, 64, P, layers=layers, max_seqs=256)
    before = [t.clone() for t in (cache.k_codes, cache.k_scale, cache.v_codes, cache.v_scale)]
    tables = ints(rows, cuda)
    out, info = cache.compact(tables, ints(lengths, cuda))
    cache.check()
    want, move = ref.compact(rows, lengths, P)
    assert out.tolist() == want
    held = {x for r in want for x in r if x >= 0}
    assert info.tolist() == [len(held), pages - len(held), len(move), 0] and (not held or max(held) == len(held) - 1)
    for t, b in zip((cache.k_codes, cache.k_scale, cache.v_codes, cache.v_scale), before):
        for src, dst in move.items():
            b[:, dst] = b[:, src]
        assert torch.equal(t, b)
    again, info = cache.compact(out, ints(lengths, cuda), out_tables=out)  # in place; nothing left to move
    assert again.tolist() == want and info[2] == 0


def test_compact_unusable_tables_are_handed_on(cuda):
    cache = make_cache(cuda, 9, 1, 64, 16)
    rows = [[8, 12, -1], [3, -1, 5]]
    out, info = cache.compact(ints(rows, cuda), ints([20, 10], cuda))
    with pytest.raises(RuntimeError):
        cache.check()
    assert out.tolist() == rows and info[2] == 0


def test_fork_and_compact_in_a_graph(cuda):
    """The page moves launch as dependents of the table kernels: the same inside a capture."""
    import torch
    import kv_reference as ref
    from ffn_residual_mesh_b200.graphs import StepGraph
    P = 16
    cache = make_cache(cuda, 60, 2, 64, P, layers=2)
    rows, lengths = [[40, 3, 59, -1, -1], [50, 7, -1, -1, -1]], [40, 20]
    tables, lens = ints(rows, cuda), ints(lengths, cuda)
    parents, extra = ints([0, 1, 0], cuda), ints([1, 1, 1], cuda)
    t2, l2 = torch.empty(3, 5, dtype=torch.int32, device=cuda), torch.empty(3, dtype=torch.int32, device=cuda)
    t3, info, info3 = torch.empty_like(t2), ints([0] * 4, cuda), ints([0] * 4, cuda)

    def step():
        cache.fork(tables, lens, parents, extra, out_tables=t2, out_lengths=l2, info=info)
        cache.compact(t2, l2, out_tables=t3, info=info3)

    graph = StepGraph(step)
    parents.copy_(ints([1, 0, 1], cuda))
    before = cache.k_codes.clone()
    graph.replay()
    torch.cuda.synchronize()
    cache.check()
    want, want_len, copies = ref.fork(rows, lengths, [1, 0, 1], [1, 1, 1], 60, P, 5)
    assert t2.tolist() == want and l2.tolist() == want_len
    packed, move = ref.compact(want, want_len, P)
    assert t3.tolist() == packed
    for pairs in (copies, move.items()):
        for src, dst in pairs:
            before[:, dst] = before[:, src]
    assert torch.equal(cache.k_codes, before)
    graph.close()


def test_copy_pages(cuda):
    import torch
    cache = make_cache(cuda, 9, 3, 128, 32, layers=2)
    before = [t.clone() for t in (cache.k_codes, cache.k_scale, cache.v_codes, cache.v_scale)]
    cache.copy_pages(ints([1, 2, 1], cuda), ints([5, 0, 8], cuda))
    cache.check()
    for t, b in zip((cache.k_codes, cache.k_scale, cache.v_codes, cache.v_scale), before):
        b[:, [5, 0, 8]] = b[:, [1, 2, 1]]
        assert torch.equal(t, b)
    cache.copy_pages(ints([1, 9], cuda), ints([-1, 2], cuda))  # neither fits the pool
    with pytest.raises(RuntimeError):
        cache.check()
    assert torch.equal(cache.k_codes, before[0])


def test_forked_samples_continue_alone(cuda):
    """fork, append to each child, attend: every child sees its own tokens after the shared ones."""
    import torch
    import kv_reference as ref
    H, G, D, P = 2, 4, 64, 16
    cache = make_cache(cuda, 40, H, D, P, seed=2)
    rows, lengths = [[7, 3, -1, -1], [1, 2, 9, -1]], [21, 40]
    g = torch.Generator(device=cuda).manual_seed(0)
    tables, lens = ints(rows, cuda), ints(lengths, cuda)
    for step in range(20):
        parents = [0, 0, 1, 1, 0] if step == 0 else [0, 1, 2, 3, 4]
        tables, lens, _ = cache.fork(tables, lens, ints(parents, cuda), ints([1] * 5, cuda))
        x = torch.randn(5, H * (G + 2), D, device=cuda, generator=g).half()
        cache.append(0, x[:, :H], x[:, H:2 * H], tables, lens)
        out = cache.attend(0, x[:, 2 * H:], tables, lens)
    cache.check()
    t = tables.tolist()
    assert lens.tolist() == [41, 41, 60, 60, 41]
    opened = [r[n // P] if n % P else r[n // P - 1] for r, n in zip(t, lens.tolist())]
    assert len(set(opened)) == 5
    want, mag, _ = ref.attend(x[:, 2 * H:], cache.k_codes[0], cache.k_scale[0], cache.v_codes[0], cache.v_scale[0], t, lens.tolist(),
                              [0, 1, 2, 3, 4, 5])
    assert ((out.double() - want).abs() <= 2.0 ** -11 * want.abs() + (2.0 ** -11 + 2.0 ** -13) * mag + 1e-6).all()


# ---------------------------------------------------------------------------------- refusals
def test_arguments_are_refused(cuda):
    import torch
    from ffn_residual_mesh_b200.kvcache import PagedKvCache, RotaryTable, rotary
    cache = make_cache(cuda, 4, 2, 64, 16)
    t, n = ints([[0, 1], [2, 3]], cuda), ints([5, 20], cuda)
    q, k = torch.randn(2, 4, 64, device=cuda).half(), torch.randn(2, 2, 64, device=cuda).half()
    table = rope_table(64, 64, cuda)
    st = ints([0, 1, 2], cuda)
    bad = [
        lambda: cache.attend(1, q, t, n), lambda: cache.attend(-1, q, t, n),
        lambda: cache.attend(0, q.float(), t, n), lambda: cache.attend(0, q.double(), t, n),
        lambda: cache.attend(0, q[:, :3], t, n), lambda: cache.attend(0, q[..., :32], t, n),
        lambda: cache.attend(0, q[:1], t, n), lambda: cache.attend(0, q[0], t, n),
        lambda: cache.attend(0, q, t.long(), n), lambda: cache.attend(0, q, t, n.long()),
        lambda: cache.attend(0, q, t, n[:1]), lambda: cache.attend(0, q, t.t(), n), lambda: cache.attend(0, q, t[0], n),
        lambda: cache.attend(0, q, t, n, starts=st[:2]), lambda: cache.attend(0, q, t, n, out=q.float()),
        lambda: cache.attend(0, q, t, n, out=q[:1]), lambda: cache.attend(0, q, t, n, out=q[:1].expand(2, 4, 64)),
        lambda: cache.attend(0, q, t, n, lse=torch.empty(2, 3, device=cuda)), lambda: cache.attend(0, q, t, n, window=-1),
        lambda: cache.attend(0, q, t, n, scale=0.0), lambda: cache.attend(0, q, t, n, scale=math.nan),
        lambda: cache.attend(0, q, t, n, scale=math.inf), lambda: cache.attend(0, q.cpu(), t, n),
        lambda: cache.attend(0, q.permute(0, 2, 1).contiguous().permute(0, 2, 1), t, n),
        lambda: cache.append(0, k, k.float(), t, n), lambda: cache.append(0, k, k[:1], t, n),
        lambda: cache.append(0, k[:, :1], k, t, n), lambda: cache.append(2, k, k, t, n), lambda: cache.append(0, k, k, t, n, q=q),
        lambda: cache.append(0, k, k, t, n, rope=table, q=q.float()), lambda: cache.append(0, k[:1], k[:1], t, n),
        lambda: cache.append(0, k, k, t, n, rope=rope_table(64, 66, cuda)), lambda: cache.append(0, k, k, t, n.cpu()),
        lambda: cache.read(0, t, n, None, 3), lambda: cache.read(0, t, n, st, 2, dtype=torch.int8),
        lambda: cache.fork(t, n, ints([0], cuda), ints([0, 1], cuda)), lambda: cache.fork(t, n, ints([0], cuda), ints([0], cuda), out_tables=t[:1]),
        lambda: cache.fork(t, n, ints([0] * 65, cuda), ints([0] * 65, cuda)),
        lambda: cache.compact(t, n[:1]), lambda: cache.compact(t.long(), n), lambda: cache.copy_pages(t, t),
        lambda: cache.copy_pages(ints([0], cuda), ints([1, 2], cuda)), lambda: cache.copy_pages(ints([0] * 5, cuda), ints([1] * 5, cuda)),
        lambda: rotary(q, ints([0], cuda), table), lambda: rotary(q, ints([0, 1], cuda).long(), table),
        lambda: rotary(q[..., :32], ints([0, 1], cuda), table), lambda: rotary(q, ints([0, 1], cuda), table, out=q.float()),
        lambda: rotary(q, ints([0, 1], cuda), table, out=q[:1].expand(2, 4, 64)),
        lambda: PagedKvCache(1, 4, 2, 96), lambda: PagedKvCache(1, 4, 2, 64, page_tokens=48), lambda: PagedKvCache(0, 4, 2, 64),
        lambda: PagedKvCache(1, 5, 2, 64, page_tokens=16, buffers=(cache.k_codes, cache.v_codes, cache.k_scale, cache.v_scale)),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was accepted")
    cache.check()


def test_empty_batches(cuda):
    import torch
    from ffn_residual_mesh_b200.kvcache import rotary
    cache = make_cache(cuda, 4, 2, 64, 16)
    none, q = ints([], cuda), torch.empty(0, 4, 64, device=cuda).half()
    t0 = torch.empty(0, 3, dtype=torch.int32, device=cuda)
    assert cache.attend(0, q, t0, none).shape == (0, 4, 64)
    cache.append(0, q[:, :2], q[:, :2], t0, none)
    assert cache.read(0, t0, none, None, 0)[0].shape == (0, 2, 64)
    assert rotary(q, none, rope_table(4, 64, cuda)).shape == (0, 4, 64)
    tables, lens, info = cache.fork(t0, none, none, none)
    assert info.tolist() == [0, 4, 0, 0]
    tables, info = cache.compact(t0, none)
    assert info.tolist() == [0, 4, 0, 0]
    cache.copy_pages(none, none)
    # sequences, but no rows
    out = cache.attend(0, q, ints([[0], [1]], cuda), ints([3, 0], cuda), starts=ints([0, 0, 0], cuda))
    assert out.shape == (0, 4, 64)
    cache.check()
