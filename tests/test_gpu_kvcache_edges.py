"""The paged cache where its data is unusual: scales of zero and of no use, table entries that name no
page, padded rows, overlapping memory, other streams, autograd.

Attention is held to the bounds of test_gpu_kvcache.py: the output's rounding, 2^-11 + 2^-13 of
sum p|v| and 1e-6; lse to 2e-5 of max(1, |lse|).
"""
from __future__ import annotations

import math

import pytest

from test_gpu_kvcache import check_attend, ints, make_cache, rope_table, row_starts

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------------------------- scales
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("zero", [0.0, -0.0, 1e-44, 1e-30])
def test_value_scales_of_zero_keep_their_weight(cuda, dtype, D, zero):
    """A block whose value scale is zero (or too small for f32's reciprocals) holds values of zero: its keys
    keep their share of the softmax. On tiles with and without masked keys, whatever its codes."""
    def some(cache, rows, q):
        for row in rows:
            for page in row[:8:2]:
                cache.v_scale[0, page] = zero
            cache.v_scale[0, row[4], 0] = 0.5  # one head of a page only
    check_attend(cuda, [1, 1, 1], [333, 40, 256], 2, 4, D, 32, dtype, seed=D, tamper=some, with_starts=False)
    check_attend(cuda, [5, 300, 130], [400, 512, 300], 2, 4, D, 32, dtype, seed=D, tamper=some)
    check_attend(cuda, [200], [700], 1, 4, D, 64, dtype, seed=D, tamper=some, causal=False)


def test_value_scales_of_zero_everywhere(cuda):
    def none(cache, rows, q):
        cache.v_scale.zero_()
    def both(cache, rows, q):
        cache.v_scale.zero_()
        cache.k_scale.zero_()
    for tamper in (none, both):
        check_attend(cuda, [1, 1], [300, 17], 2, 4, 128, 32, seed=1, tamper=tamper, with_starts=False)
        check_attend(cuda, [300, 20], [300, 600], 2, 4, 128, 32, "bf16", seed=1, tamper=tamper)


def test_value_scales_far_apart(cuda):
    """Zero blocks beside small, ordinary and large ones in one row."""
    def uneven(cache, rows, q):
        for row in rows:
            for i, s in enumerate((0.0, 1e-18, 1e-12, 1e-3, 30.0, 0.0)):
                cache.v_scale[0, row[i]] = s
    check_attend(cuda, [1, 60], [300, 300], 2, 4, 128, 32, seed=8, tamper=uneven)
    check_attend(cuda, [280], [400], 2, 4, 128, 32, "bf16", seed=8, tamper=uneven)


@pytest.mark.parametrize("which", ["k_scale", "v_scale"])
@pytest.mark.parametrize("value", [-0.02, -math.inf, math.inf])
def test_scales_of_no_use_count_as_nan(cuda, which, value):
    """A scale is finite and not negative; any other marks its block as a NaN does, in both kernels."""
    import torch
    tables, lengths = ints([[0, 1, 2, 3, 4, 5], [6, 7, 8, 9, 10, 11]], cuda), ints([300, 384], cuda)
    for new in ([1, 1], [250, 130]):
        got = []
        for bad in (value, math.nan):
            cache = make_cache(cuda, 12, 2, 128, 64, seed=3)
            getattr(cache, which)[0, 1, 1] = bad  # tokens 64..127 of sequence 0, kv head 1
            q = torch.randn(sum(new), 8, 128, device=cuda, generator=torch.Generator(device=cuda).manual_seed(1)).half()
            lse = torch.empty(sum(new), 8, device=cuda)
            got.append((cache.attend(0, q, tables, lengths, starts=ints(row_starts(new), cuda), lse=lse), lse))
            cache.check()
        (out, lse), (want, want_lse) = got
        assert torch.isnan(out[:new[0], 4:].float()).any() and not torch.isnan(out[:, :4]).any() and not torch.isnan(out[new[0]:]).any()
        assert torch.equal(torch.nan_to_num(out, 9.0), torch.nan_to_num(want, 9.0))
        assert torch.equal(torch.isnan(out), torch.isnan(want))
        assert torch.equal(torch.isnan(lse), torch.isnan(want_lse))


@pytest.mark.parametrize("value", [-0.02, math.inf])
def test_append_to_a_block_of_no_use_marks_it(cuda, value):
    import torch
    cache = make_cache(cuda, 3, 2, 64, 16)
    cache.k_scale[0, 1, 0] = value
    cache.v_scale[0, 1, 1] = value
    x = torch.randn(1, 2, 64, device=cuda)
    cache.append(0, x, x, ints([[0, 1]], cuda), ints([20], cuda))
    cache.check()
    assert torch.isnan(cache.k_scale[0, 1]).tolist() == [True, False]
    assert torch.isnan(cache.v_scale[0, 1]).tolist() == [False, True]

# ---------------------------------------------------------------------------------- tables
@pytest.mark.parametrize("entry", [-1, -2, -3, -2 ** 31, 12, 2 ** 31 - 1])
@pytest.mark.parametrize("new,G", [([1, 1], 4), ([3, 2], 4), ([90, 1], 4), ([130, 150], 8), ([180], 4)])
def test_table_entries_that_name_no_page_are_skipped(cuda, entry, new, G):
    """Whatever the entry, in either kernel: recorded, its keys left out, the others weighed as ever."""
    import torch
    import kv_reference as ref
    H, D, P = 2, 128, 32
    cache = make_cache(cuda, 12, H, D, P, seed=4)
    rows, lengths = [[3, 7, 0, 11, 5, 1, 9], [2, 4, 6, 8, 10, 3, 7]][:len(new)], [220, 224][:len(new)]
    q = torch.randn(sum(new), H * G, D, device=cuda, generator=torch.Generator(device=cuda).manual_seed(2)).half()
    starts = row_starts(new)
    broken = [list(r) for r in rows]
    broken[0][0] = entry  # before every new token: the others see what the sequence without that page has
    lse = torch.empty(sum(new), H * G, device=cuda)
    out = cache.attend(0, q, ints(broken, cuda), ints(lengths, cuda), starts=ints(starts, cuda), lse=lse)
    with pytest.raises(RuntimeError, match="page id"):
        cache.check()
    cache.check()
    less, short = [r[1:] if i == 0 else r for i, r in enumerate(rows)], [lengths[0] - P] + lengths[1:]
    want, mag, want_lse = ref.attend(q, cache.k_codes[0], cache.k_scale[0], cache.v_codes[0], cache.v_scale[0], less, short, starts)
    if new[0] > short[0]:
        raise AssertionError("the page must lie before the new tokens")
    assert ((out.double() - want).abs() <= 2.0 ** -11 * want.abs() + (2.0 ** -11 + 2.0 ** -13) * mag + 1e-6).all()
    assert ((lse.double() - want_lse).abs() <= 2e-5 * want_lse.abs().clamp(min=1)).all()


def test_a_table_of_no_pages_gives_zeros(cuda):
    import torch
    cache = make_cache(cuda, 4, 2, 128, 32)
    for n in (1, 200):
        q = torch.randn(n, 8, 128, device=cuda).half()
        lse = torch.zeros(n, 8, device=cuda)
        out = cache.attend(0, q, ints([[-2] * 8], cuda), ints([250], cuda), starts=ints([0, n], cuda), lse=lse)
        with pytest.raises(RuntimeError, match="page id"):
            cache.check()
        assert (out == 0).all() and (lse == -math.inf).all()


# ---------------------------------------------------------------------------------- fork in place
@pytest.mark.parametrize("n", [6, 33, 700, 2500])
def test_fork_writes_lengths_in_place(cuda, n):
    """out_lengths on the input lengths, parents in any order: the same as apart from them."""
    import numpy as np
    import torch
    rng = np.random.default_rng(n)
    P, width = 16, 5
    lengths = rng.integers(0, 3 * P, n)
    rows, at = [], 0
    for x in lengths:
        k = -(-int(x) // P)
        rows.append([*range(at, at + k), *[-1] * (width - k)])
        at += k
    parents = rng.permutation(n)
    parents[rng.integers(0, n, n // 5)] = int(parents[0])
    extra = rng.integers(0, P, n)
    cache = make_cache(cuda, at + 4 * n, 1, 64, P, max_seqs=n)
    args = [ints(v, cuda) for v in (rows, lengths.tolist(), parents.tolist(), extra.tolist())]
    tables, lens, info = cache.fork(*args)
    cache.check()
    assert lens.tolist() == (lengths[parents] + extra).tolist()
    for place in (1, 2, 3):  # on the lengths, the parents, the room
        own = [a.clone() for a in args]
        got, out, got_info = cache.fork(*own, out_lengths=own[place])
        cache.check()
        assert out.data_ptr() == own[place].data_ptr()
        assert torch.equal(got, tables) and torch.equal(out, lens) and torch.equal(got_info, info)
    buffer = torch.cat([args[1], ints([0] * 8, cuda)])  # shifted by some
    got, out, _ = cache.fork(args[0], buffer[:n], *args[2:], out_lengths=buffer[5:n + 5])
    cache.check()
    assert torch.equal(got, tables) and torch.equal(out, lens)


def test_fork_short_of_pages_in_place(cuda):
    """Nothing is forked: zeros where out_lengths lies, be it the input."""
    cache = make_cache(cuda, 3, 1, 64, 16)
    tables, lengths, extra = ints([[0, 1, 2, -1]], cuda), ints([40], cuda), ints([16], cuda)
    for out in (None, lengths):
        _, lens, info = cache.fork(tables, lengths, ints([0], cuda), extra, out_lengths=out)
        with pytest.raises(MemoryError):
            cache.check()
        assert lens.tolist() == [0] and info.tolist() == [3, 0, 0, 1] and lengths.tolist() == [40 if out is None else 0]


def test_page_tables_on_one_another_are_refused(cuda):
    import torch
    cache = make_cache(cuda, 40, 1, 64, 16)
    buffer = torch.zeros(64, dtype=torch.int32, device=cuda)
    n, p, e = ints([5, 20], cuda), ints([0, 1], cuda), ints([1, 1], cuda)
    t = buffer[:6].view(2, 3)
    for call in (lambda: cache.fork(t, n, p, e, out_tables=t), lambda: cache.fork(t, n, p, e, out_tables=buffer[5:11].view(2, 3)),
                 lambda: cache.fork(t, n, p, e, out_tables=buffer[10:16].view(2, 3), out_lengths=buffer[15:17]),
                 lambda: cache.fork(t, n, p, e, out_tables=buffer[10:16].view(2, 3), info=buffer[7:11]),
                 lambda: cache.fork(t, n, p, e, out_lengths=buffer[20:22], info=buffer[21:25]),
                 lambda: cache.compact(t, n, out_tables=buffer[3:9].view(2, 3)), lambda: cache.compact(t, n, info=buffer[5:9], out_tables=t)):
        with pytest.raises(ValueError):
            call()
    cache.fork(t, n, p, e, out_tables=buffer[6:12].view(2, 3), out_lengths=buffer[12:14], info=buffer[14:18])  # side by side
    cache.check()


def test_fork_that_asks_for_more_than_2_to_the_31_pages(cuda):
    """The children's wishes add up past 32 bits: short of pages, nothing changed."""
    import torch
    n, width = 2049, 1 << 20
    cache = make_cache(cuda, 3, 1, 64, 16, max_seqs=n)
    before = cache.k_codes.clone()
    out = torch.empty(n, width, dtype=torch.int32, device=cuda)
    tables, lens, info = cache.fork(ints([[0, 1]], cuda), ints([20], cuda), ints([0] + [-1] * (n - 1), cuda),
                                    torch.full((n,), 16 * width - 32, dtype=torch.int32, device=cuda), out_tables=out)
    with pytest.raises(MemoryError):
        cache.check()
    assert (lens == 0).all() and info.tolist() == [2, 1, 0, 2 ** 31 - 1]
    assert (tables[:: 512] == -1).all() and torch.equal(cache.k_codes, before)


# ---------------------------------------------------------------------------------- memory that overlaps
def test_overlapping_outputs_are_refused(cuda):
    import torch
    from ffn_residual_mesh_b200.kvcache import rotary
    H, G, D, T = 2, 4, 64, 6
    cache = make_cache(cuda, 8, H, D, 16)
    tables, lengths, starts = ints([[0, 1], [2, 3]], cuda), ints([20, 9], cuda), ints([0, 4, 6], cuda)
    table, pos = rope_table(64, D, cuda), ints([0, 1, 2, 3, 4, 5], cuda)
    qkv = torch.randn(T + 1, H * G + 2 * H + 1, D, device=cuda).half()
    q, k, v = qkv[:T, :H * G], qkv[:T, H * G:H * G + H], qkv[:T, H * G + H:H * G + 2 * H]
    flat, args = qkv.flatten(), dict(starts=starts, rope=table, q=q)
    before = [t.clone() for t in (qkv, cache.k_codes, cache.v_codes)]
    for call in (lambda: rotary(q, pos, table, out=qkv[:T, 1:H * G + 1]), lambda: rotary(q, pos, table, out=qkv[1:, :H * G]),
                 lambda: rotary(q, pos, table, out=flat[:T * H * G * D].view(T, H * G, D)),
                 lambda: rotary(q, pos, table, out=torch.empty(999 * D, device=cuda).half().as_strided((T, H * G, D), (D, D, 1))),
                 lambda: cache.append(0, k, v, tables, lengths, q_out=qkv[:T, 2:H * G + 2], **args),
                 lambda: cache.append(0, k, v, tables, lengths, q_out=qkv[:T, H + 1:H * G + H + 1], **args),
                 lambda: cache.append(0, k, qkv[:T, :H].clone(), tables, lengths, q_out=qkv[:T, 2 * H:H * G + 2 * H], **dict(args, q=q.clone())),
                 lambda: cache.attend(0, q, tables, lengths, starts=starts, out=qkv[:T, 1:H * G + 1]),
                 lambda: cache.attend(0, q, tables, lengths, starts=starts, out=qkv[1:, :H * G]),
                 lambda: cache.attend(0, q, tables, lengths, starts=starts, lse=flat.view(torch.float32)[:T * H * G].view(T, H * G))):
        with pytest.raises(ValueError):
            call()
    cache.check()
    for a, b in zip(before, (qkv, cache.k_codes, cache.v_codes)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("new", [[1, 1], [5, 3], [150, 90]])
def test_in_place_and_in_a_packed_row(cuda, new):
    """q rotated and attended in place, and into another slice of its own packed row: as into memory apart."""
    import torch
    from ffn_residual_mesh_b200.kvcache import rotary
    H, G, D = 2, 4, 128
    T, lengths = sum(new), ints([200, 90], cuda)
    tables, starts = ints([[*range(13)], [*range(13, 26)]], cuda), ints(row_starts(new), cuda)
    table = rope_table(256, D, cuda)
    packed = torch.randn(T, 2 * H * G + 2 * H, D, device=cuda, generator=torch.Generator(device=cuda).manual_seed(1)).half()

    def step(q, out, k, v):
        cache = make_cache(cuda, 26, H, D, 16, seed=1)
        got = cache.append(0, k, v, tables, lengths, starts=starts, rope=table, q=q, q_out=out)
        rotated = got.clone()
        seen = cache.attend(0, got, tables, lengths, starts=starts, out=out)
        cache.check()
        return rotated, seen

    def parts(x):
        return x[:, :H * G], x[:, H * G:2 * H * G], x[:, 2 * H * G:2 * H * G + H], x[:, 2 * H * G + H:]

    q, _, k, v = parts(packed.clone())
    want = step(q, torch.empty_like(q), k, v)
    q, spare, k, v = parts(packed.clone())
    got = step(q, spare, k, v)
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and torch.equal(q, packed[:, :H * G])
    q, _, k, v = parts(packed.clone())
    got = step(q, q, k, v)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    x = packed.clone()
    pos = torch.arange(T, device=cuda).int()
    rotary(x[:, :H], pos, table, out=x[:, H:2 * H])
    assert torch.equal(x[:, H:2 * H], rotary(packed[:, :H], pos, table)) and torch.equal(x[:, 2 * H:], packed[:, 2 * H:])

# ---------------------------------------------------------------------------------- rows of no sequence
@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_read_pads_with_zeros(cuda, dtype):
    """Rows before starts[0] and from starts[seqs] on read as zeros, as they do in append and attend."""
    import torch
    cache = make_cache(cuda, 4, 2, 64, 16)
    tables, lengths = ints([[0, 1], [2, 3]], cuda), ints([20, 9], cuda)
    kind = {"f16": torch.float16, "f32": torch.float32}[dtype]
    want = cache.read(0, tables, lengths, ints([0, 3, 5], cuda), 5, dtype=kind)
    got = cache.read(0, tables, lengths, ints([2, 5, 7], cuda), 11, dtype=kind)
    cache.check()
    for g, w in zip(got, want):
        assert torch.equal(g[2:7], w) and (g[:2] == 0).all() and (g[7:] == 0).all()
    cache.read(0, tables, ints([20, 1], cuda), ints([0, 3, 5], cuda), 5)  # more rows than tokens: still recorded
    with pytest.raises(RuntimeError):
        cache.check()


def test_append_pads_with_zeros(cuda):
    """The same rows in append: no token is taken from them, and their queries become zeros."""
    import torch
    tables, lengths = ints([[0, 1], [2, 3]], cuda), ints([20, 9], cuda)
    table, x = rope_table(32, 64, cuda), torch.randn(11, 2, 64, device=cuda).half()
    caches = [make_cache(cuda, 4, 2, 64, 16) for _ in range(2)]
    q = caches[0].append(0, x, x, tables, lengths, starts=ints([2, 5, 7], cuda), rope=table, q=x)
    want = caches[1].append(0, x[2:7], x[2:7], tables, lengths, starts=ints([0, 3, 5], cuda), rope=table, q=x[2:7])
    for c in caches:
        c.check()
    assert torch.equal(q[2:7], want) and (q[:2] == 0).all() and (q[7:] == 0).all()
    assert torch.equal(caches[0].k_codes, caches[1].k_codes) and torch.equal(caches[0].v_scale, caches[1].v_scale)


def test_rows_of_no_sequence_are_refused(cuda):
    """With no sequence at all there is nothing that the outputs could be."""
    import torch
    cache = make_cache(cuda, 4, 2, 64, 16)
    t0, none, start = torch.empty(0, 3, dtype=torch.int32, device=cuda), ints([], cuda), ints([0], cuda)
    x = torch.randn(5, 2, 64, device=cuda).half()
    for call in (lambda: cache.read(0, t0, none, start, 5), lambda: cache.append(0, x, x, t0, none, starts=start, rope=rope_table(8, 64, cuda), q=x),
                 lambda: cache.attend(0, x, t0, none, starts=start)):
        with pytest.raises(ValueError):
            call()
    cache.append(0, x, x, t0, none, starts=start)  # nothing to write, nothing to return
    cache.check()


# ---------------------------------------------------------------------------------- autograd
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("inverse", [False, True])
def test_rotary_gradient_through_autograd(cuda, dtype, interleaved, inverse):
    """The gradient is the other direction's rotation of the output's, bit for bit; also of a sum (an expanded
    gradient), of a packed row, of one head shared by several, and twice."""
    import torch
    from test_gpu_kvcache import types
    from ffn_residual_mesh_b200.kvcache import rotary
    kind, table = types()[dtype], rope_table(40, 32, cuda, interleaved)
    pos = ints([0, 7, 39, 7, 1], cuda)
    g = torch.Generator(device=cuda).manual_seed(2)
    x = torch.randn(5, 6, 48, device=cuda, generator=g).to(kind).requires_grad_()
    w = torch.randn(5, 3, 48, device=cuda, generator=g).to(kind)
    y = rotary(x[:, 1:4], pos, table, inverse=inverse)
    assert y.requires_grad and torch.equal(y.detach(), rotary(x.detach()[:, 1:4], pos, table, inverse=inverse))
    (got,) = torch.autograd.grad(y, x, w)
    assert torch.equal(got[:, 1:4], rotary(w, pos, table, inverse=not inverse)) and (got[:, 0] == 0).all() and (got[:, 4:] == 0).all()
    ones = torch.ones_like(w)
    (got,) = torch.autograd.grad(rotary(x[:, 1:4], pos, table, inverse=inverse).sum(), x)
    assert torch.equal(got[:, 1:4], rotary(ones, pos, table, inverse=not inverse))
    shared = torch.randn(5, 1, 48, device=cuda, generator=g).requires_grad_()
    (got,) = torch.autograd.grad(rotary(shared.expand(5, 3, 48), pos, table, inverse=inverse), shared, w.float())
    want = rotary(w.float(), pos, table, inverse=not inverse).double().sum(1, keepdim=True)
    assert ((got.double() - want).abs() <= 3 * 2.0 ** -23 * (1 + want.abs()) * 4).all()
    v = w.clone().requires_grad_()  # linear in the output's gradient too
    (first,) = torch.autograd.grad(rotary(x[:, 1:4], pos, table, inverse=inverse), x, v, create_graph=True)
    (second,) = torch.autograd.grad(first, v, torch.ones_like(first))
    assert torch.equal(second, rotary(ones, pos, table, inverse=inverse))


def test_rotary_gradient_against_differences(cuda):
    import torch
    from ffn_residual_mesh_b200.kvcache import rotary
    table, pos = rope_table(40, 16, cuda), ints([3, 39], cuda)
    g = torch.Generator(device=cuda).manual_seed(4)
    x = torch.randn(2, 2, 20, device=cuda, generator=g).requires_grad_()

    def loss(z):  # a smooth function of the rotated values, in 64 bits behind the kernel
        return (rotary(z, pos, table).double() ** 3).sum()

    (got,) = torch.autograd.grad(loss(x), x)
    with torch.no_grad():
        for t, h, d in ((0, 0, 0), (0, 1, 7), (1, 0, 8), (1, 1, 15), (1, 1, 19)):
            step = torch.zeros_like(x)
            step[t, h, d] = 2.0 ** -7
            diff = (loss(x + step) - loss(x - step)).item() / 2.0 ** -6
            # f32 rounding of values up to 5 (3 y^2 <= 75 of 2^-22 each, over the step) and the cube's third derivative
            assert abs(diff - got[t, h, d].item()) <= 40 * 75 * 2.0 ** -22 * 64 + 2.0 ** -14 * 4 + 1e-5 * abs(diff)


def test_rotary_into_memory_and_autograd(cuda):
    import torch
    from ffn_residual_mesh_b200.kvcache import rotary
    table, pos = rope_table(8, 16, cuda), ints([1, 2], cuda)
    x = torch.randn(2, 2, 16, device=cuda).requires_grad_()
    for bad in (dict(out=torch.empty(2, 2, 16, device=cuda)), dict(out=x)):
        with pytest.raises(ValueError):
            rotary(x, pos, table, **bad)
    with pytest.raises(ValueError):
        rotary(x.detach(), pos, table, out=torch.empty(2, 2, 16, device=cuda, requires_grad=True))
    with torch.no_grad():
        y = rotary(x, pos, table)
        assert not y.requires_grad and torch.equal(rotary(x, pos, table, out=torch.empty_like(y)), y)
    with torch.inference_mode():
        z = x.detach().clone()
        assert torch.equal(rotary(z, pos, table, out=z), y)


def test_outputs_that_are_given_count_as_written(cuda):
    """Their version moves, so that autograd does not take a saved tensor for what it was."""
    import torch
    from ffn_residual_mesh_b200.kvcache import rotary
    cache, table = make_cache(cuda, 8, 2, 64, 16), rope_table(64, 64, cuda)
    tables, lengths = ints([[0, 1], [2, 3]], cuda), ints([20, 9], cuda)
    q, k = torch.randn(2, 4, 64, device=cuda).half(), torch.randn(2, 2, 64, device=cuda).half()
    out, lse = torch.empty_like(q), torch.empty(2, 4, device=cuda)
    t2, l2, info = torch.empty_like(tables), torch.empty_like(lengths), ints([0] * 4, cuda)
    two = ints([0, 1], cuda)
    for call, given in ((lambda: rotary(q, two, table, out=out), (out,)),
                        (lambda: cache.append(0, k, k, tables, lengths, rope=table, q=q, q_out=out), (out,)),
                        (lambda: cache.attend(0, q, tables, lengths, out=out, lse=lse), (out, lse)),
                        (lambda: cache.fork(tables, lengths, two, two, out_tables=t2, out_lengths=l2, info=info), (t2, l2, info)),
                        (lambda: cache.compact(tables, lengths, out_tables=t2, info=info), (t2, info))):
        before = [x._version for x in (*given, q, k, tables, lengths)]
        call()
        after = [x._version for x in (*given, q, k, tables, lengths)]
        assert [b > a for a, b in zip(before, after)] == [True] * len(given) + [False] * 4
    scale = torch.ones_like(q, requires_grad=True)
    y = scale * out  # saves out
    cache.attend(0, q, tables, lengths, out=out)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    with torch.inference_mode():
        cache.attend(0, q, tables, lengths, out=torch.empty_like(q))
        cache.attend(0, q, tables, lengths, out=out)
    inside = None
    with torch.inference_mode():
        inside = torch.empty_like(q)
    cache.attend(0, q, tables, lengths, out=inside)
    assert torch.equal(inside, out)
    cache.check()


# ---------------------------------------------------------------------------------- another stream
def test_arguments_may_be_dropped_while_another_stream_works(cuda):
    """The side stream is kept busy for some 50 ms; what the calls read there is dropped on the current one and
    its memory asked for again."""
    import torch
    from ffn_residual_mesh_b200.kvcache import RotaryTable, rotary
    H, G, D, T = 4, 8, 128, 64
    rows = [[2 * i, 2 * i + 1] for i in range(T)]
    lengths = [3 + i % 29 for i in range(T)]

    def work(stream, drop):
        """q's and k's rotation, append, attend, read, fork, compact; every argument made here."""
        cache = make_cache(cuda, 2 * T + 8, H, D, 16, max_seqs=T, seed=1)
        g = torch.Generator(device=cuda).manual_seed(3)
        q, k = (torch.randn(T, n, D, device=cuda, generator=g).half() for n in (H * G, H))
        t, n, pos = ints(rows, cuda), ints(lengths, cuda), ints(lengths, cuda)
        table, starts = rope_table(64, D, cuda), ints(list(range(T + 1)), cuda)
        parents, extra = ints(list(range(T))[::-1], cuda), ints([1] * T, cuda)
        lse = torch.empty(T, H * G, device=cuda)
        if stream is not None:
            stream.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(stream):
                torch.cuda._sleep(100_000_000)
        r = rotary(q, pos, table, stream=stream)
        a = cache.append(0, k, k, t, n, starts=starts, rope=table, q=q, stream=stream)
        o = cache.attend(0, q, t, n, starts=starts, lse=lse, stream=stream)
        back = cache.read(0, t, n, starts, T, stream=stream)
        f = cache.fork(t, n, parents, extra, stream=stream)
        c = cache.compact(t, n, stream=stream)
        if drop:
            size = [x.shape for x in (q, k, t, n, pos, starts, parents, table.cos_sin)]
            kind = [x.dtype for x in (q, k, t, n, pos, starts, parents, table.cos_sin)]
            del q, k, t, n, pos, starts, parents, extra, table
            again = [torch.full(s, 3, dtype=d, device=cuda) for s, d in zip(size, kind) for _ in range(3)]
            torch.cuda.current_stream().synchronize()
            del again
        if stream is not None:
            stream.synchronize()
        cache.check(stream)
        return [r, a, o, lse, *back, *f, *c, cache.k_codes, cache.k_scale, cache.v_codes]

    want = work(None, False)
    got = work(torch.cuda.Stream(), True)
    for i, (x, y) in enumerate(zip(got, want)):
        assert torch.equal(x, y), i


@pytest.mark.parametrize("value", [1e18, 1e36, 9e37, 3e38])
def test_value_scales_up_to_the_largest(cuda, value):
    """Codes of -1, 0 and 1 under scales up to f32's largest: also those whose reciprocal is a subnormal."""
    def large(cache, rows, q):
        cache.v_codes.clamp_(-1, 1)
        cache.v_scale.fill_(value)
    check_attend(cuda, [1, 1], [300, 17], 2, 4, 128, 32, "bf16", seed=1, tamper=large, with_starts=False)
    check_attend(cuda, [300, 20], [300, 600], 2, 4, 128, 32, "bf16", seed=1, tamper=large)
    check_attend(cuda, [200], [256], 1, 4, 256, 64, "bf16", seed=1, tamper=large, causal=False)


# ---------------------------------------------------------------------------------- strides that count for nothing
def test_strides_of_single_rows_and_heads_do_not_matter(cuda):
    """One token or one head: its stride is never used, so it may be anything."""
    import torch
    from ffn_residual_mesh_b200.kvcache import rotary
    cache, table = make_cache(cuda, 4, 1, 64, 16), rope_table(64, 64, cuda)
    flat = torch.randn(4096, device=cuda).half()
    tables, one, two = ints([[0, 1]], cuda), ints([20], cuda), ints([[0, 1], [2, 3]], cuda)
    q = flat[:4 * 64].view(1, 4, 64)
    odd = flat.as_strided((1, 4, 64), (301, 64, 1))
    assert torch.equal(cache.attend(0, odd, tables, one), cache.attend(0, q, tables, one))
    out = torch.zeros(4096, device=cuda).half().as_strided((1, 4, 64), (333, 64, 1))
    assert torch.equal(cache.attend(0, q, tables, one, out=out), cache.attend(0, q, tables, one))
    tall = flat.as_strided((2, 1, 64), (64, 37, 1))
    lengths = ints([20, 9], cuda)
    assert torch.equal(cache.attend(0, tall, two, lengths), cache.attend(0, tall.contiguous(), two, lengths))
    z = flat.clone().as_strided((1, 4, 64), (7, 64, 1))
    assert torch.equal(rotary(z, one, table, out=z.as_strided((1, 4, 64), (99, 64, 1))), rotary(q, one, table))
    cache.check()


def test_fork_and_compact_of_the_largest_pool_and_batch(cuda):
    """2^20 pages and 4096 sequences: the most shared memory that the table kernels take."""
    import numpy as np
    import kv_reference as ref
    rng, P, n, pages, width = np.random.default_rng(3), 16, 4096, 1 << 20, 4
    lengths = rng.integers(0, 40, n).tolist()
    ids, at, rows = rng.permutation(pages), 0, []
    for x in lengths:
        k = -(-x // P)
        rows.append([*ids[at:at + k].tolist(), *[-1] * (width - k)])
        at += k
    cache = make_cache(cuda, pages, 1, 64, P, max_seqs=n)
    parents, extra = rng.integers(-1, n, n).tolist(), rng.integers(0, 20, n).tolist()
    tables, lens, info = cache.fork(ints(rows, cuda), ints(lengths, cuda), ints(parents, cuda), ints(extra, cuda))
    packed, count = cache.compact(tables, lens)
    cache.check()
    want, want_len, copies = ref.fork(rows, lengths, parents, extra, pages, P, width)
    assert tables.tolist() == want and lens.tolist() == want_len and info[2] == len(copies)
    want, move = ref.compact(want, want_len, P)
    assert packed.tolist() == want and count[2] == len(move)
