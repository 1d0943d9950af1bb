"""Rotary positions, the paged K/V cache, attention over a shared prefix and draft verification against plain 64-bit
implementations, at the sizes and masks where they can go wrong."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

import genref as R
from zillaphp_b200 import native
from zillaphp_b200.backend import B200Backend
from zillaphp_b200.kv import PagedKv

pytestmark = pytest.mark.gpu


@pytest.fixture
def bufs():
    b = R.Buffers(B200Backend())
    yield b
    b.be.sync()
    assert native.load().zilla_check_device() == 0, native.last_error()
    b.close()


def starts(new):
    return [0] + list(np.cumsum(new).tolist())


def i32(x):
    return torch.tensor(x, dtype=torch.int32)


# ---------------------------------------------------------------------------------------- rotary positions
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("rows,heads,dim,rot,interleaved,scaling,inverse,off,ld,far", [
    (1, 1, 2, 2, 0, 0, 0, 0, 0, 10),                  # the smallest
    (1, 4, 32, 32, 0, 0, 0, 0, 0, 128),
    (5, 3, 128, 64, 1, 3, 0, 8, 512, 1 << 20),        # part of the head, by parts, packed rows
    (9, 2, 80, 26, 0, 1, 1, 3, 175, 1000),            # odd halves and offsets: one element at a time
    (9, 2, 80, 28, 1, 1, 1, 2, 180, 1000),            # two at a time
    (33, 5, 96, 88, 1, 2, 1, 4, 600, (1 << 31) - 1),  # four at a time, the farthest positions
    (700, 40, 128, 128, 0, 0, 0, 0, 0, 131072),       # several rows a block
    (17, 2, 256, 256, 1, 0, 1, 0, 0, 5),
    (2500, 7, 64, 56, 0, 3, 0, 0, 0, 4096),
])
def test_rope(bufs, dtype, rows, heads, dim, rot, interleaved, scaling, inverse, off, ld, far):
    g = torch.Generator().manual_seed(rows + rot)
    wide = heads * dim
    ld = ld or wide
    x = torch.randn((rows, ld), generator=g).to(R.DT[dtype])
    pos = torch.randint(-min(far, 100), far, (rows,), generator=g, dtype=torch.int64).to(torch.int32)
    pos[0] = far if far < 2 ** 31 else far - 1
    args = (10000.0, scaling, 8.0, 4096, 1.0, 32.0)
    table = bufs.new(rot + 2)
    bufs.be.ropeTableDev(table, rot, *args)
    before = torch.randn((rows, wide + 8), generator=g).to(R.DT[dtype])
    ix, iy, ip = bufs.put(x), bufs.put(before), bufs.put(pos)
    bufs.be.ropeDev(ix, off, ld, iy, 4 if ld == wide else 0, wide + 8, ip, table, R.CODE[dtype], rows, heads, dim, rot, interleaved, inverse)
    y = bufs.get(iy, before.shape, R.DT[dtype])
    y_off = 4 if ld == wide else 0
    ref, size = R.rotate(x[:, off:off + wide].reshape(rows, heads, dim), pos, rot, interleaved, R.rates(rot, *args), -1.0 if inverse else 1.0)
    got = y[:, y_off:y_off + wide].reshape(rows, heads, dim).double()
    tol = size * (R.ROTATION + R.far(pos)) + (R.half_step(ref, R.DT[dtype]) if dtype != "fp32" else 0)
    assert ((got - ref).abs() <= tol).all(), float(((got - ref).abs() - tol).max())
    assert torch.equal(got[..., rot:], ref[..., rot:])                       # copied bit for bit
    keep = torch.ones(wide + 8, dtype=torch.bool)
    keep[y_off:y_off + wide] = False
    assert torch.equal(y[:, keep], before[:, keep])                         # nothing else is written


def test_rope_in_place_in_a_packed_row(bufs):
    g = torch.Generator().manual_seed(3)
    x = torch.randn((37, 6 * 64), generator=g)
    pos = torch.arange(37, dtype=torch.int32)
    table = bufs.new(66)
    bufs.be.ropeTableDev(table, 64)
    ix, ip = bufs.put(x), bufs.put(pos)
    bufs.be.ropeDev(ix, 128, 384, ix, 128, 384, ip, table, 0, 37, 2, 64, 64)
    y = bufs.get(ix, x.shape, torch.float32)
    ref, size = R.rotate(x[:, 128:256].reshape(37, 2, 64), pos, 64, 0, R.rates(64))
    assert ((y[:, 128:256].reshape(37, 2, 64).double() - ref).abs() <= size * R.ROTATION).all()
    assert torch.equal(y[:, :128], x[:, :128]) and torch.equal(y[:, 256:], x[:, 256:])


def test_rope_gradient_against_differences(bufs):
    """The inverse turn is the gradient: central differences of f(x) = sum(w y(x)), linear in x, so that the step adds
    only rounding (fp32 y: 2^-24 of about 4 each, over 16 elements and a step of 0.5)."""
    g = torch.Generator().manual_seed(4)
    rows, dim, rot = 2, 8, 6
    x, w, pos = torch.randn((rows, 1, dim), generator=g), torch.randn((rows, 1, dim), generator=g), i32([3, 70000])
    table = bufs.new(rot + 2)
    bufs.be.ropeTableDev(table, rot, 10000.0, 3, 4.0, 64)
    ip, iy = bufs.put(pos), bufs.new(x.numel())

    def turn(t, inverse):
        bufs.be.ropeDev(bufs.put(t), 0, dim, iy, 0, dim, ip, table, 0, rows, 1, dim, rot, 1, inverse)
        return bufs.get(iy, t.shape, torch.float32).double()

    grad = turn(w, 1)
    for r in range(rows):
        for i in range(dim):
            e = torch.zeros_like(x)
            e[r, 0, i] = 0.5
            d = ((turn(x + e, 0) - turn(x - e, 0)) * w.double()).sum()
            assert abs(float(d) - float(grad[r, 0, i])) < 16 * 4 * 2.0 ** -23 / 0.5


# ---------------------------------------------------------------------------------------- the cache
def batch_of(new, length, prefix, page, seed, max_pages=0, spare=3):
    """start, pages, prefix pages and the number of pages, in no order."""
    g = torch.Generator().manual_seed(seed)
    most = max(max_pages, max(1, -(-max(list(length) + [1]) // page)))
    first = max(1, -(-prefix // page))
    order = torch.randperm(first + most * len(new) + spare, generator=g).to(torch.int32)
    return starts(new), order[first:first + most * len(new)].reshape(len(new), most), order[:first], order.numel(), most


@pytest.mark.parametrize("src,dtype", [("fp32", "bf16"), ("bf16", "bf16"), ("fp32", "fp16"), ("fp16", "fp16")])
@pytest.mark.parametrize("new,length,hq,hk,dim,rot,interleaved,page,prefix,packed,pad", [
    ([1], [1], 4, 4, 32, 32, 0, 16, 0, False, 0),
    ([1, 0, 3], [17, 0, 16], 6, 2, 64, 24, 1, 16, 5, True, 2),        # a sequence without rows, rows behind the last
    ([5, 2], [5, 130], 7, 1, 128, 128, 0, 128, 999999, False, 1),
    ([40, 1, 300], [40, 64, 301], 8, 8, 128, 96, 1, 64, 70, True, 0),  # prompts, pages crossed
    ([3], [70], 0, 2, 64, 64, 0, 32, 0, False, 0),                    # no queries
    ([2, 2], [9, 3], 2, 1, 32, 0, 0, 16, 0, True, 0),                 # no rotation
    ([2] * 300, [33] * 300, 2, 1, 32, 30, 0, 32, 3, False, 4),        # more sequences than threads
    ([0, 1, 3, 0] * 700, [5] * 2800, 2, 1, 32, 32, 0, 16, 3, True, 3), # more than a block looks through one by one
])
def test_append(bufs, src, dtype, new, length, hq, hk, dim, rot, interleaved, page, prefix, packed, pad):
    start, pages, _, count, most = batch_of(new, length, 0, page, 5)
    rows = start[-1] + pad
    g = torch.Generator().manual_seed(6)
    wide = (hq + 2 * hk) * dim
    ld = wide + 24
    x = torch.randn((max(rows, 1), ld), generator=g).to(R.DT[src])
    q, k, v = x[:, 8:8 + hq * dim], x[:, 8 + hq * dim:8 + (hq + hk) * dim], x[:, 8 + (hq + hk) * dim:8 + wide]
    kv = PagedKv(count, page, hk, dim, dtype)
    shape = (count, hk, page, dim)
    kc, vc = (torch.randn(shape, generator=g).to(R.DT[dtype]) for _ in range(2))
    bufs.write(kv.k_id, kc)
    bufs.write(kv.v_id, vc)
    out = torch.randn((rows, max(hq, 1), dim), generator=g).to(R.DT[dtype])
    table = 0
    if rot:
        table = bufs.new(rot + 2)
        bufs.be.ropeTableDev(table, rot)
    io = bufs.put(out)
    if packed:
        i = bufs.put(x)
        inputs = (i, 8, ld, i, 8 + hq * dim, ld, i, 8 + (hq + hk) * dim, ld)
    else:
        inputs = (bufs.put(q) if hq else 0, 0, hq * dim, bufs.put(k), 0, hk * dim, bufs.put(v), 0, hk * dim)
    kv.append(R.CODE[src], *inputs, io if hq else 0, bufs.put(i32(start)), bufs.put(i32(length)), bufs.put(pages), len(new), rows, hq,
              most, prefix, table, rot, interleaved)
    at = torch.tensor([length[b] - new[b] + j for b in range(len(new)) for j in range(new[b])], dtype=torch.long)
    own = torch.tensor([b for b in range(len(new)) for _ in range(new[b])], dtype=torch.long)
    n, T = start[-1], R.DT[dtype]
    plan, pos = R.rates(rot) if rot else None, at + prefix
    got = bufs.get(io, out.shape, T)
    if hq:
        ref, size = R.rotate(q[:n].reshape(n, hq, dim), pos, rot, interleaved, plan or ([], 1.0))
        tol = size * (R.ROTATION + R.far(pos)) + R.half_step(ref, T)
        assert ((got[:n].double() - ref).abs() <= tol).all()
        assert torch.equal(got[n:], out[n:])
    page_of, slot = pages[own, at // page].long(), at % page
    ref, size = R.rotate(k[:n].reshape(n, hk, dim), pos, rot, interleaved, plan or ([], 1.0))
    got_k, got_v = bufs.get(kv.k_id, shape, T), bufs.get(kv.v_id, shape, T)
    tol = size * (R.ROTATION + R.far(pos)) + R.half_step(ref, T)
    assert ((got_k[page_of, :, slot].double() - ref).abs() <= tol).all()
    vc[page_of, :, slot] = v[:n].reshape(n, hk, dim).to(T)
    assert torch.equal(got_v, vc)                                    # values rounded once, nothing else written
    got_k[page_of, :, slot] = kc[page_of, :, slot]
    assert torch.equal(got_k, kc)
    kv.close()


# ---------------------------------------------------------------------------------------- attention
def run_attend(bufs, dtype, new, length, hq, hk, dim, page, prefix, pad=0, max_new=0, max_len=0, scale=None, max_pages=0, seed=7,
               junk=True, sharp=1.5, repeat=1, only=None):
    T = R.DT[dtype]
    start, pages, front, count, most = batch_of(new, length, prefix, page, seed, max_pages)
    rows = start[-1] + pad
    g = torch.Generator().manual_seed(seed)
    shape = (count, hk, page, dim)
    k, v = (torch.randn(shape, generator=g).to(T) for _ in range(2))
    kj, vj = k.clone(), v.clone()
    if junk:   # every slot that no sequence holds: NaN, infinities
        held = torch.zeros((count, page), dtype=torch.bool)
        for i in range(prefix):
            held[front[i // page], i % page] = True
        for b, n in enumerate(length):
            for i in range(n):
                held[pages[b, i // page], i % page] = True
        bad = torch.tensor([float("nan"), float("inf"), float("-inf")]).to(T)
        m = ~held[:, None, :, None].expand(shape)
        kj[m] = bad[torch.arange(int(m.sum())) % 3]
        vj[m] = bad[torch.arange(int(m.sum())) % 3]
    q = (torch.randn((rows, hq, dim), generator=g) * sharp).to(T)
    out = torch.randn((rows, hq, dim), generator=g).to(T)
    kv = PagedKv(count, page, hk, dim, dtype)
    bufs.write(kv.k_id, kj)
    bufs.write(kv.v_id, vj)
    max_new, max_len = max_new or max(max(new), 1), max_len or max(length)
    scale = 1 / math.sqrt(dim) if scale is None else scale
    work = kv.attend_work(len(new), rows, hq, prefix, max_new, max_len)
    io = bufs.put(out)
    iw = bufs.new(work) if work else 0
    if work:   # whatever the workspace holds does not matter
        bufs.be.bufferUpload(iw, np.full(work, np.nan, np.float32))
    args = (bufs.put(q), io, bufs.put(i32(start)), bufs.put(i32(length)), bufs.put(pages), bufs.put(front), len(new), rows, hq, most,
            prefix, max_new, max_len, scale, iw)
    kv.attend(*args)
    got = bufs.get(io, out.shape, T)
    for _ in range(repeat - 1):   # the same bits every time: a copy that overtakes a read shows here
        bufs.be.zeroDev(io, max(1, out.numel() // 2))
        kv.attend(*args)
        again = bufs.get(io, out.shape, T)
        assert torch.equal(again[:start[-1]], got[:start[-1]]), (again[:start[-1]] != got[:start[-1]]).nonzero()[:8].tolist()
        got[start[-1]:] = again[start[-1]:] = out[start[-1]:]
    if only is not None:          # the reference for some sequences alone, their rows moved together
        keep = [t for b in only for t in range(start[b], start[b + 1])]
        q, got, out = q[keep], got[keep], out[keep]
        start, length, pages = starts([new[b] for b in only]), [length[b] for b in only], pages[only]
    ref = R.attend(q, k, v, start, length, pages.tolist(), front.tolist(), prefix, scale, page)
    n = start[-1]
    tol = R.attend_tolerance(ref, dim, T)
    assert torch.isfinite(got[:n]).all()
    err = (got[:n].double() - ref[0][:n]).abs()
    assert (err <= tol[:n]).all(), float((err / tol[:n]).max())
    assert torch.equal(got[n:], out[n:])
    kv.close()


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("dim", [32, 64, 128])
@pytest.mark.parametrize("new,length,hq,hk,page,prefix,pad", [
    ([1], [1], 1, 1, 16, 0, 0),                              # one key: the smallest
    ([1], [1], 1, 1, 16, 1, 0),
    ([1, 0, 2], [1, 0, 64], 3, 1, 16, 15, 2),                # a sequence without rows, an odd group
    ([1, 1, 1], [65, 63, 17], 4, 4, 64, 64, 0),              # a key past a stage, MHA
    ([5, 1, 3], [200, 129, 3], 8, 2, 128, 130, 1),           # drafts, pages that end inside a stage
    ([2, 4], [513, 40], 7, 1, 32, 0, 0),                     # no prefix, joined slots
    ([6] * 5, [6, 70, 33, 100, 64], 16, 2, 32, 257, 3),      # more rows than one tile of 32
    ([30, 1], [90, 20], 8, 2, 16, 40, 0),                    # a prompt in the middle: several row tiles
    ([1, 2], [0, 1], 4, 2, 16, 33, 0),                       # rows in front of the first own key: the prefix alone
])
def test_attend(bufs, dtype, dim, new, length, hq, hk, page, prefix, pad):
    run_attend(bufs, dtype, new, length, hq, hk, dim, page, prefix, pad)


def test_attend_large_batches(bufs):
    """More sequences than a block of the join looks through one by one, empty ones among them."""
    run_attend(bufs, "bf16", [0, 1, 0, 2] * 400, [i % 40 + 2 for i in range(1600)], 2, 1, 32, 16, 300, 3, only=list(range(0, 1600, 7)) + [1599])
    run_attend(bufs, "fp16", [0] * 1200 + [3] + [0] * 1300, [3] * 2501, 4, 2, 64, 16, 700, 1)


def test_attend_rows_without_keys(bufs):
    run_attend(bufs, "bf16", [2, 1, 3], [0, 5, 1], 4, 2, 64, 16, 0, 1)       # joined or direct: zeros
    run_attend(bufs, "bf16", [1, 2], [0, 0], 4, 2, 64, 16, 0, max_len=16)
    run_attend(bufs, "fp16", [3, 1], [1, 400], 4, 2, 64, 16, 0)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_attend_loose_bounds(bufs, dtype):
    """max_new and max_len far above what is there."""
    run_attend(bufs, dtype, [1, 3], [20, 300], 8, 2, 128, 16, 100, 1, max_new=9, max_len=1000, max_pages=80)


@pytest.mark.parametrize("max_new", [2 ** 31 - 1, 2 ** 30 + 1, 2 ** 26])
def test_attend_largest_bound_of_new_rows(bufs, max_new):
    """Row tiles are counted from the rows that are there, also where max_new times the group passes 31 bits."""
    run_attend(bufs, "bf16", [3, 1, 40], [20, 300, 90], 64, 1, 32, 16, 100, 1, max_new=max_new)


@pytest.mark.parametrize("dtype,dim,hq,hk,page,prefix,new,longest", [
    ("bf16", 32, 4, 4, 16, 96, [1] * 16, 32), ("fp16", 64, 8, 2, 16, 5, [2, 1, 0, 3], 64), ("bf16", 128, 24, 1, 128, 65, [1, 3], 100),
    ("fp16", 128, 4, 2, 32, 130, [4] * 230, 90),          # a prefix in front of many sequences' own keys
    ("bf16", 64, 16, 2, 64, 256, [5, 1] * 120, 70), ("bf16", 128, 3, 3, 16, 1, [2, 1] * 90, 257), ("bf16", 32, 40, 1, 16, 63, [1] * 4, 0)])
def test_attend_short_prefix(bufs, dtype, dim, hq, hk, page, prefix, new, longest):
    """Short prefixes: each block runs over the prefix and its sequence's own keys, no parts are joined."""
    length = [min(longest, n + (37 * i) % (longest + 1)) for i, n in enumerate(new)]
    run_attend(bufs, dtype, new, length, hq, hk, dim, page, prefix, 2, max_len=max(longest, 1), max_pages=-(-max(longest, 1) // page))


@pytest.mark.parametrize("dtype,dim,hq,hk,page,prefix,new,longest", [
    ("bf16", 128, 32, 8, 64, 0, 5, 2048), ("bf16", 128, 32, 8, 16, 0, 3, 1500), ("fp16", 64, 16, 8, 32, 0, 3, 2048), ("bf16", 128, 32, 8, 128, 0, 1, 2000),
    ("bf16", 64, 32, 4, 64, 0, 5, 1800), ("fp16", 32, 16, 8, 16, 0, 2, 2000), ("bf16", 128, 32, 8, 64, 3000, 5, 2048), ("fp16", 64, 32, 4, 16, 2500, 4, 900)])
def test_attend_long_replies_repeat(bufs, dtype, dim, hq, hk, page, prefix, new, longest):
    """A full machine: 96 sequences with long replies, eight runs alike to the bit, some sequences against 64 bits."""
    length = [max(new, longest - 137 * i % longest) for i in range(96)]
    run_attend(bufs, dtype, [new] * 96, length, hq, hk, dim, page, prefix, repeat=8, only=[0, 41, 95], junk=False)


def test_attend_scales(bufs):
    run_attend(bufs, "bf16", [1, 2], [100, 70], 4, 2, 64, 16, 90, scale=-0.3)
    run_attend(bufs, "bf16", [1, 2], [100, 70], 4, 2, 64, 16, 90, scale=0.0)
    run_attend(bufs, "bf16", [1, 2], [100, 70], 4, 2, 64, 16, 90, scale=0.4, sharp=8.0)   # one key takes nearly all


@pytest.mark.parametrize("dtype,dim,hq,hk,prefix,new", [
    ("bf16", 128, 32, 8, 1000, [1] * 33), ("fp16", 64, 32, 4, 777, [3, 1, 5, 2] * 4), ("bf16", 32, 4, 4, 300, [1] * 130),
    ("bf16", 128, 5, 1, 129, [2] * 60), ("fp16", 128, 16, 2, 2049, [4] * 9),
    ("bf16", 128, 32, 8, 2500, [4] * 70), ("fp16", 32, 66, 1, 128, [1]), ("bf16", 64, 130, 2, 1, [3, 1]), ("fp16", 128, 28, 4, 640, [6] * 40)])
def test_attend_many_rows_behind_one_prefix(bufs, dtype, dim, hq, hk, prefix, new):
    length = [n + (7 * i) % 90 for i, n in enumerate(new)]
    run_attend(bufs, dtype, new, length, hq, hk, dim, 64, prefix, 2)


def test_attend_many_rows_scales(bufs):
    for scale, sharp in ((-0.2, 1.5), (0.0, 1.5), (0.4, 8.0)):
        run_attend(bufs, "bf16", [2] * 20, [20] * 20, 8, 1, 64, 16, 700, scale=scale, sharp=sharp)


@pytest.mark.parametrize("dtype,dim,hq,hk,page,prefix,new,longest", [
    ("bf16", 128, 64, 8, 16, 1, [5] * 22, 300), ("fp16", 128, 64, 8, 64, 63, [5] * 22, 270),     # less than a step, less than a tile
    ("bf16", 64, 128, 8, 32, 127, [4] * 20, 300), ("fp16", 64, 128, 8, 128, 129, [4] * 21, 400),   # about a tile
    ("bf16", 32, 64, 16, 16, 257, [3, 0, 1] * 20, 500),                                            # rows that end in a first stream
    ("fp16", 32, 256, 8, 64, 200, [1, 2] * 9, 600), ("bf16", 128, 17, 1, 64, 900, [2] * 13, 90),   # fewer tiles than blocks, an odd group
    ("fp16", 128, 3, 1, 16, 8000, [6], 70), ("bf16", 64, 24, 3, 128, 4100, [1] * 3, 40)])          # 18 and 24 rows
def test_attend_prefix_and_replies(bufs, dtype, dim, hq, hk, page, prefix, new, longest):
    """Prefixes that are enough work for a kernel of their own beside the sequences' own keys."""
    length = [max(n, longest - 61 * i % longest) for i, n in enumerate(new)]
    run_attend(bufs, dtype, new, length, hq, hk, dim, page, prefix, 2)


def test_attend_long_prefix_scales(bufs):
    for scale, sharp in ((-0.2, 1.5), (0.0, 1.5), (0.4, 8.0)):
        run_attend(bufs, "fp16", [2] * 20, [20] * 20, 16, 2, 64, 16, 2800, scale=scale, sharp=sharp)


def test_attend_bad_numbers_are_recorded():
    """A page number outside the cache counts as keys and values of zero; a length beyond the call's leaves its rows alone."""
    b = R.Buffers(B200Backend())
    kv = PagedKv(4, 16, 1, 32, "bf16")
    ones = torch.ones((4, 1, 16, 32), dtype=torch.bfloat16)
    b.write(kv.k_id, ones)
    b.write(kv.v_id, ones)
    q, out = torch.ones((2, 1, 32)).to(torch.bfloat16), torch.full((2, 1, 32), 7.0).to(torch.bfloat16)
    io = b.put(out)
    for page in (4, -1, 2 ** 31 - 1, -2 ** 31):
        kv.attend(b.put(q), io, b.put(i32([0, 1, 2])), b.put(i32([16, 999])), b.put(i32([[page], [0]])), 0, 2, 2, 1, 1, 0, 1, 16, 1.0,
                  b.new(max(1, kv.attend_work(2, 2, 1, 0, 1, 16))))
        got = b.get(io, out.shape, torch.bfloat16)
        assert (got[0] == 0).all() and (got[1] == 7).all()
        assert native.load().zilla_check_device() == -3
        assert native.load().zilla_check_device() == 0
    table, x = b.new(34), b.put(torch.ones((2, 32)))
    b.be.ropeTableDev(table, 32)
    kv.append(0, x, 0, 32, x, 0, 32, x, 0, 32, io, b.put(i32([0, 1, 2])), b.put(i32([1, 17])), b.put(i32([[9], [0]])), 2, 2, 1, 1, 0, table, 32)
    assert native.load().zilla_check_device() == -3            # a bad page, and a token behind the table's end
    assert torch.equal(b.get(kv.k_id, ones.shape, torch.bfloat16), ones) and torch.equal(b.get(io, out.shape, torch.bfloat16), got)
    kv.close()
    b.close()


# ---------------------------------------------------------------------------------------- verification
def rows_of(new, vocab, ld, seed, near=0.7):
    g = np.random.default_rng(seed)
    rows = sum(new)
    z = g.standard_normal((rows, vocab)) * 2
    e = np.exp(z)
    p = np.zeros((rows, ld), np.float32)
    q = np.zeros((rows, ld), np.float32)
    p[:, :vocab] = e / e.sum(1, keepdims=True)
    e = np.exp(z + g.standard_normal((rows, vocab)) * near)
    q[:, :vocab] = e / e.sum(1, keepdims=True)
    draft = np.array([g.choice(vocab, p=(r[:vocab].astype(np.float64) / r[:vocab].astype(np.float64).sum())) for r in q], np.int32).reshape(-1)
    return p, q, draft, g.random(rows, np.float32)


def run_verify(bufs, p, q, draft, u, new, vocab, pad=0):
    start, rows, ld = starts(new), p.shape[0], p.shape[1]
    before = np.full(rows + pad, -7, np.int32)
    it, ia = bufs.put(torch.from_numpy(before)), bufs.put(torch.full((len(new),), -7, dtype=torch.int32))
    zeros = np.zeros((pad, ld), np.float32)
    bufs.be.draftVerifyDev(bufs.put(torch.from_numpy(np.concatenate([p, zeros]))), ld,
                           0 if q is None else bufs.put(torch.from_numpy(np.concatenate([q, zeros]))), ld,
                           bufs.put(torch.from_numpy(np.concatenate([draft, np.zeros(pad, np.int32)]))),
                           bufs.put(torch.from_numpy(np.concatenate([u, np.zeros(pad, np.float32)]))), bufs.put(i32(start)), it, ia,
                           len(new), rows + pad, vocab)
    tokens, accepted = R.verify(p, q, draft, u, start, vocab)
    got = bufs.get(it, (rows + pad,), torch.int32).tolist()
    assert bufs.get(ia, (len(new),), torch.int32).tolist() == accepted
    assert got[:rows] == [tokens[i] for i in range(rows)] and got[rows:] == [-7] * pad
    return accepted


@pytest.mark.parametrize("vocab,ld", [(1, 1), (2, 4), (65, 65), (129, 132), (4096, 4096), (5001, 5003), (33333, 33336), (131072, 131072)])
@pytest.mark.parametrize("certain", [False, True])
def test_verify(bufs, vocab, ld, certain):
    for seed, new in enumerate(([1], [5, 1, 0, 9, 2], [3] * 40 if vocab < 6000 else [4] * 6)):
        p, q, draft, u = rows_of(new, vocab, ld, seed)
        run_verify(bufs, p, None if certain else q, draft, u, new, vocab, 2)


@pytest.mark.parametrize("vocab,ld,batch", [(517, 517, 1500), (2100, 2100, 950), (25000, 25003, 500), (9000, 9000, 160)])
def test_verify_many_sequences(bufs, vocab, ld, batch):
    """More sequences than the machine holds at once, and about as many."""
    new = [(1, 2, 3, 0)[b % 4] for b in range(batch)]
    p, q, draft, u = rows_of(new, vocab, ld, 21)
    run_verify(bufs, p, q, draft, u, new, vocab, 1)


def test_verify_borders(bufs):
    """Equal probabilities, numbers of 0 and next to 1, every draft taken, none taken, over 32 drafts."""
    new = [40, 40, 3]
    p, q, draft, u = rows_of(new, 300, 300, 11, near=0.0)
    q[:] = p
    u[:] = np.float32(1 - 2.0 ** -24)
    assert run_verify(bufs, p, q, draft, u, new, 300) == [39, 39, 2]        # u q < p for every u < 1
    u[35] = 0.0
    p[35, draft[35]] = 0.0                                                   # 0 < 0 fails: the 36th draft
    q[45] *= np.float32(1.5)                                                 # the 6th of the second
    u[39] = u[79] = u[82] = 0.0
    assert run_verify(bufs, p, q, draft, u, new, 300) == [35, 5, 2]
    u[39] = u[79] = u[82] = np.float32(1.0)                                  # above every border: the last with a weight
    run_verify(bufs, p, q, draft, u, new, 300)


def test_verify_degenerate_rows(bufs):
    """No residual, zeros throughout, NaN, negative and infinite values."""
    new = [2, 2, 2, 2, 1]
    p, q, draft, u = rows_of(new, 50, 50, 12)
    q[0] = np.float32(2.0) * p[0] + 1                # fails, nothing left: drawn from p
    p[2] = 0.0                                       # fails, and no weight at all: token 0
    p[4, 10:20] = np.nan
    p[4, draft[4]] = 0.0
    p[6, draft[6]] = 0.0
    p[6, 5] = -1.0
    u[0] = u[4] = u[6] = 0.9
    run_verify(bufs, p, q, draft, u, new, 50)


def test_verify_bad_drafts_are_recorded():
    b = R.Buffers(B200Backend())
    new = [3, 2]
    p, q, draft, u = rows_of(new, 40, 40, 13)
    u[:] = 0.0
    draft[1], draft[3] = 40, -2 ** 31
    assert run_verify(b, p, q, draft, u, new, 40) == [1, 0]
    assert native.load().zilla_check_device() == -3
    it, ia = b.put(torch.full((5,), -7, dtype=torch.int32)), b.put(i32([9, 9]))
    b.be.draftVerifyDev(b.put(torch.from_numpy(p)), 40, 0, 0, b.put(torch.from_numpy(draft)), b.put(torch.from_numpy(u)), b.put(i32([0, 6, 5])),
                        it, ia, 2, 5, 40)                                      # rows that do not fit
    assert b.get(ia, (2,), torch.int32).tolist() == [0, 0] and b.get(it, (5,), torch.int32).tolist() == [-7] * 5
    assert native.load().zilla_check_device() == -3
    b.close()


# ---------------------------------------------------------------------------------------- together
class Loop:
    """Generation steps as a program runs them: a shared prompt, then rounds of drafted tokens for every sequence."""

    def __init__(self, bufs, dtype="bf16", hq=8, hk=2, dim=64, page=16, prefix=37, size=5, most=4, seed=21):
        self.b, self.dtype, self.hq, self.hk, self.dim, self.page, self.prefix, self.size, self.most = bufs, dtype, hq, hk, dim, page, prefix, size, most
        self.rows, self.max_len, self.vocab = size * most, 96, 65
        self.g = torch.Generator().manual_seed(seed)
        self.wide = (hq + 2 * hk) * dim
        own_pages, front = self.max_len // page, -(-prefix // page)
        order = torch.randperm(own_pages * size + front, generator=self.g).to(torch.int32)
        self.front, self.pages = order[:front], order[front:].reshape(size, own_pages)
        self.kv = PagedKv(order.numel(), page, hk, dim, dtype)
        self.table = bufs.new(dim + 2)
        bufs.be.ropeTableDev(self.table, dim)
        self.ids = {n: bufs.new(w) for n, w in (("x", self.rows * self.wide), ("q", self.rows * hq * dim), ("out", self.rows * hq * dim),
                                                 ("start", size + 1), ("len", size), ("draft", self.rows), ("u", self.rows), ("p", self.rows * 65),
                                                 ("tokens", self.rows), ("accepted", size), ("logits", self.rows * 65), ("head", hq * dim * 65))}
        self.ids["pages"], self.ids["front"] = bufs.put(self.pages), bufs.put(self.front)
        self.ids["work"] = bufs.new(max(1, self.kv.attend_work(size, self.rows, hq, prefix, most, self.max_len)))
        self.k_ref = torch.zeros((order.numel(), hk, page, dim), dtype=R.DT[dtype])
        self.v_ref = self.k_ref.clone()
        x = torch.randn((prefix, self.wide), generator=self.g)
        i = bufs.put(x)
        self.kv.append(0, 0, 0, 0, i, hq * dim, self.wide, i, (hq + hk) * dim, self.wide, 0, bufs.put(i32([0, prefix])), bufs.put(i32([prefix])),
                       self.ids["front"], 1, prefix, 0, front, 0, self.table, dim)
        self.store(x, torch.arange(prefix), self.front[torch.arange(prefix) // page].long(), torch.arange(prefix) % page)
        self.length = [0] * size

    def store(self, x, pos, page_of, slot):
        n, a, c = x.shape[0], self.hq * self.dim, (self.hq + self.hk) * self.dim
        k, _ = R.rotate(x[:, a:c].reshape(n, self.hk, self.dim), pos, self.dim, 0, R.rates(self.dim))
        self.k_ref[page_of, :, slot] = k.to(self.k_ref.dtype)
        self.v_ref[page_of, :, slot] = x[:, c:].reshape(n, self.hk, self.dim).to(self.k_ref.dtype)

    def new_step(self, new):
        """Uploads one step's inputs."""
        self.new, self.start = new, starts(new)
        self.length = [a + n for a, n in zip(self.length, new)]
        self.x = torch.randn((self.rows, self.wide), generator=self.g)
        self.draft = torch.randint(0, self.vocab, (self.rows,), generator=self.g, dtype=torch.int32)
        self.u = torch.rand((self.rows,), generator=self.g)
        logits = torch.randn((self.rows, self.vocab), generator=self.g)
        for name, t in (("x", self.x), ("start", i32(self.start)), ("len", i32(self.length)), ("draft", self.draft), ("u", self.u), ("logits", logits)):
            self.b.write(self.ids[name], t)

    def calls(self):
        d, i, hq, hk = self.dim, self.ids, self.hq, self.hk
        self.kv.append(0, i["x"], 0, self.wide, i["x"], hq * d, self.wide, i["x"], (hq + hk) * d, self.wide, i["q"], i["start"], i["len"], i["pages"],
                       self.size, self.rows, hq, self.pages.shape[1], self.prefix, self.table, d)
        self.kv.attend(i["q"], i["out"], i["start"], i["len"], i["pages"], i["front"], self.size, self.rows, hq, self.pages.shape[1], self.prefix,
                       self.most, self.max_len, 1 / math.sqrt(d), i["work"])
        self.b.be.softmaxRowsFwdDev(i["logits"], i["p"], self.rows, self.vocab)
        self.b.be.draftVerifyDev(i["p"], self.vocab, 0, 0, i["draft"], i["u"], i["start"], i["tokens"], i["accepted"], self.size, self.rows, self.vocab)

    def check(self):
        n, T = self.start[-1], R.DT[self.dtype]
        own = torch.tensor([b for b in range(self.size) for _ in range(self.new[b])], dtype=torch.long)
        at = torch.tensor([self.length[b] - self.new[b] + j for b in range(self.size) for j in range(self.new[b])], dtype=torch.long)
        self.store(self.x[:n], at + self.prefix, self.pages[own, at // self.page].long(), at % self.page)
        # attention on the cache and queries as the device holds them: their own roundings are the append's test
        q = self.b.get(self.ids["q"], (self.rows, self.hq, self.dim), T)
        k, v = (self.b.get(i, self.k_ref.shape, T) for i in (self.kv.k_id, self.kv.v_id))
        assert torch.equal(v, self.v_ref)
        # a key's rounding may fall to the other side of a border that the rotation's error reaches: one step
        assert ((k.double() - self.k_ref.double()).abs() <= 2.01 * R.half_step(torch.maximum(k.abs(), self.k_ref.abs()), T)).all()
        ref = R.attend(q, k, v, self.start, self.length, self.pages.tolist(), self.front.tolist(), self.prefix, 1 / math.sqrt(self.dim), self.page)
        got = self.b.get(self.ids["out"], (self.rows, self.hq, self.dim), T)
        tol = R.attend_tolerance(ref, self.dim, T)
        assert ((got[:n].double() - ref[0][:n]).abs() <= tol[:n]).all()
        p = self.b.get(self.ids["p"], (self.rows, self.vocab), torch.float32).numpy()
        tokens, accepted = R.verify(p, None, self.draft.numpy(), self.u.numpy(), self.start, self.vocab)
        got = self.b.get(self.ids["tokens"], (self.rows,), torch.int32).tolist()
        assert [got[i] for i in range(n)] == [tokens[i] for i in range(n)]
        assert self.b.get(self.ids["accepted"], (self.size,), torch.int32).tolist() == accepted
        # the refused drafts leave the cache: the next step writes over them
        self.length = [m - n + a + 1 if n else m for m, n, a in zip(self.length, self.new, accepted)]


STEPS = ([1, 4, 2, 0, 3], [4, 4, 4, 4, 4], [0, 1, 0, 2, 0], [3, 2, 1, 4, 1])


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_generation_steps(bufs, dtype):
    loop = Loop(bufs, dtype)
    for new in STEPS:
        loop.new_step(list(new))
        loop.calls()
        loop.check()
    loop.kv.close()


def test_generation_steps_captured_on_another_stream(bufs):
    """The calls captured once on a stream of the program's own and replayed for each step."""
    lib = native.load()
    loop = Loop(bufs)
    loop.new_step(list(STEPS[0]))
    loop.calls()
    loop.check()
    s = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    bufs.be.sync()
    try:
        with torch.cuda.graph(graph, stream=s):
            lib.zilla_set_stream(C.c_void_p(s.cuda_stream))
            loop.calls()
        for new in STEPS[1:]:
            loop.new_step(list(new))
            with torch.cuda.stream(s):
                graph.replay()
            loop.check()
    finally:
        lib.zilla_set_stream(None)
    loop.kv.close()


def test_two_captured_calls_with_their_own_workspaces(bufs):
    """Two graphs of the same attention, each with its workspace, in flight on two streams: bit for bit the eager results."""
    lib = native.load()
    loops = [Loop(bufs, seed=s, prefix=300, page=16) for s in (1, 2)]
    want, graphs, streams = [], [], [torch.cuda.Stream() for _ in loops]
    for loop in loops:
        loop.new_step([4, 1, 4, 2, 4])
        loop.calls()
        want.append(bufs.get(loop.ids["out"], (loop.rows, loop.hq, loop.dim), torch.bfloat16))
    bufs.be.sync()
    try:
        for loop, s in zip(loops, streams):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                lib.zilla_set_stream(C.c_void_p(s.cuda_stream))
                loop.calls()
            graphs.append(g)
        for _ in range(20):
            for g, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
    finally:
        lib.zilla_set_stream(None)
    for loop, w in zip(loops, want):
        n = loop.start[-1]
        assert torch.equal(bufs.get(loop.ids["out"], w.shape, torch.bfloat16)[:n], w[:n])
        loop.kv.close()


# ---------------------------------------------------------------------------------------- refusals with real buffers
def test_refusals_leave_everything_alone(bufs):
    be, lib = bufs.be, native.load()
    small, table, ints = bufs.new(3), bufs.new(34), bufs.put(i32([0, 1, 2, 0]))
    x, y = bufs.put(torch.ones(2, 64)), bufs.put(torch.full((2, 64), 5.0))
    be.ropeTableDev(table, 32)
    kv = PagedKv(4, 16, 2, 32, "bf16")
    other = PagedKv(4, 16, 2, 32, "fp16")

    def rope(**kw):
        a = {**dict(x=x, x_off=0, x_ld=64, y=y, y_off=0, y_ld=64, pos=ints, table=table, type=0, rows=2, heads=2, dim=32, rot=32, inter=0, inv=0), **kw}
        return lib.rope_dev(*a.values())

    for bad in (dict(x=small), dict(y=small), dict(rows=3), dict(pos=0), dict(table=small), dict(x_ld=66), dict(y_off=1, y_ld=65), dict(rot=34, dim=64, heads=1)):
        assert rope(**bad) == -1, bad

    def append(cache=kv, **kw):
        a = {**dict(type=0, q=x, q_off=0, q_ld=64, k=x, k_off=0, k_ld=64, v=x, v_off=0, v_ld=64, qout=y, start=ints, len=ints, pages=ints, batch=2, rows=2,
                    q_heads=2, max_pages=1, prefix=0, table=table, rot=32, inter=0), **kw}
        return lib.zilla_kv_append(cache.id, *a.values())

    for bad in (dict(q=small), dict(k=small), dict(v=small), dict(qout=small), dict(start=small, batch=3), dict(len=0), dict(pages=small, max_pages=2),
                dict(rows=3), dict(table=small)):
        assert append(**bad) == -1, bad
    for bad in (dict(type=1 + 1), dict(type=3), dict(q_ld=63), dict(k_off=1), dict(v_off=-1), dict(q_heads=-1), dict(max_pages=0), dict(prefix=-1), dict(rot=34),
                dict(rot=31), dict(qout=x), dict(k=kv.k_id), dict(v=kv.v_id), dict(qout=kv.k_id), dict(start=y), dict(inter=2), dict(prefix=2 ** 31 - 2)):
        assert append(**bad) == -2, bad
    assert append(cache=other, type=1) == -2           # rows of another 16-bit type than the cache's
    assert append(q=small, q_heads=0, qout=0, len=bufs.put(i32([1, 1]))) == 0     # without queries theirs are not looked at

    def attend(**kw):
        a = {**dict(q=x, out=y, start=ints, len=ints, pages=ints, front=ints, batch=2, rows=2, heads=2, max_pages=1, prefix=0, max_new=1, max_len=16,
                    scale=C.c_float(1.0), work=0), **kw}
        return lib.zilla_kv_attend(kv.id, *a.values())

    for bad in (dict(heads=3), dict(heads=0), dict(max_pages=0), dict(max_len=17), dict(max_new=0), dict(prefix=-1), dict(scale=C.c_float(math.inf)),
                dict(scale=C.c_float(math.nan)), dict(out=x), dict(out=kv.k_id), dict(out=ints), dict(rows=2 ** 30, heads=4)):
        assert attend(**bad) == -2, bad
    for bad in (dict(q=small, rows=3), dict(out=small, heads=4), dict(start=small, batch=3), dict(len=0), dict(pages=small, max_pages=2), dict(prefix=100, front=small, rows=1, work=x),
                dict(prefix=2000, front=bufs.new(125), work=small)):
        assert attend(**bad) == -1, bad
    assert attend(batch=0) == 0 and attend(rows=0, q=small, out=y) == 0

    def verify(**kw):
        a = {**dict(p=x, p_ld=64, q=0, q_ld=0, draft=ints, u=ints, start=ints, tokens=y, accepted=bufs.put(i32([9, 9])), batch=2, rows=2, vocab=64), **kw}
        return lib.draft_verify_dev(*a.values())

    for bad in (dict(p=small), dict(q=small, q_ld=64), dict(rows=3), dict(draft=0), dict(u=0), dict(start=small, batch=3), dict(tokens=0), dict(accepted=0), dict(vocab=65, p_ld=65)):
        assert verify(**bad) == -1, bad
    assert verify(batch=0) == 0
    assert torch.equal(bufs.get(y, (2, 64), torch.float32), torch.full((2, 64), 5.0))
    with pytest.raises(Exception, match="rope_dev failed"):
        be.ropeDev(small, 0, 64, y, 0, 64, ints, table, 0, 2, 2, 32, 32)
    with pytest.raises(Exception, match="zilla_kv_create failed"):
        PagedKv(4, 17, 2, 32)
    be.bufferFree(other.k_id)                           # a buffer taken away from a cache: the cache is refused, not read
    assert lib.zilla_kv_k_id(other.id) == -1 and append(cache=other) == -1
    other.close()
    kv.close()


def test_far_pages(bufs):
    """A cache whose offsets pass 32 bits: its first, middle and last pages."""
    pages, page, hk, dim, prefix = 140_000, 64, 4, 128, 200      # 4.6e9 elements of K, and of V
    kv = PagedKv(pages, page, hk, dim, "bf16")
    g = torch.Generator().manual_seed(31)
    order = [pages - 1, 0, pages // 2, pages - 2, 1, 70_001, 139_000, 131_072]
    front, own = i32(order[:4]), i32(order[4:]).reshape(2, 2)
    x = torch.randn((prefix + 100, 2 * hk * dim), generator=g).to(torch.bfloat16)
    i, shape = bufs.put(x), (prefix, hk, dim)
    none = dict(table_id=0, rot_dim=0)
    kv.append(1, 0, 0, 0, i, 0, 2 * hk * dim, i, hk * dim, 2 * hk * dim, 0, bufs.put(i32([0, prefix])), bufs.put(i32([prefix])), bufs.put(front), 1, prefix, 0, 4, 0, **none)
    rest = bufs.put(x[prefix:])
    start, length = [0, 70, 100], [70, 30]
    kv.append(1, 0, 0, 0, rest, 0, 2 * hk * dim, rest, hk * dim, 2 * hk * dim, 0, bufs.put(i32(start)), bufs.put(i32(length)), bufs.put(own), 2, 100, 0, 2, prefix, **none)
    q = torch.randn((5, 8, dim), generator=g).to(torch.bfloat16)
    io = bufs.new(5 * 8 * dim)
    work = kv.attend_work(2, 5, 8, prefix, 3, 70)
    kv.attend(bufs.put(q), io, bufs.put(i32([0, 2, 5])), bufs.put(i32(length)), bufs.put(own), bufs.put(front), 2, 5, 8, 2, prefix, 3, 70, 0.1, bufs.new(max(1, work)))
    got = bufs.get(io, (5, 8, dim), torch.bfloat16)
    small = {n: k for k, n in enumerate(order)}
    k, v = torch.zeros((8, hk, page, dim)).to(torch.bfloat16), torch.zeros((8, hk, page, dim)).to(torch.bfloat16)

    def put(table, at, row):
        k[small[int(table[at // page])], :, at % page] = x[row, : hk * dim].reshape(hk, dim)
        v[small[int(table[at // page])], :, at % page] = x[row, hk * dim:].reshape(hk, dim)

    for t in range(prefix):
        put(front, t, t)
    for b in range(2):
        for t in range(length[b]):
            put(own[b], t, prefix + start[b] + t)
    ref = R.attend(q, k, v, [0, 2, 5], length, [[small[int(n)] for n in r] for r in own], [small[int(n)] for n in front], prefix, 0.1, page)
    assert ((got.double() - ref[0]).abs() <= R.attend_tolerance(ref, dim, torch.bfloat16)).all()
    kv.close()


def test_calls_on_a_stream_of_the_program(bufs):
    """The calls enqueued on torch's stream behind torch's own work, without a synchronisation between them."""
    lib = native.load()
    loop = Loop(bufs)
    loop.new_step([4, 4, 4, 4, 4])
    bufs.be.sync()
    s = torch.cuda.Stream()
    try:
        lib.zilla_set_stream(C.c_void_p(s.cuda_stream))
        with torch.cuda.stream(s):
            a = torch.ones(4096, 4096, device="cuda")
            for _ in range(20):
                a = a @ a * 1e-4                  # the calls have to wait for this
            loop.calls()
        s.synchronize()
    finally:
        lib.zilla_set_stream(None)
    loop.check()
    loop.kv.close()


# ---------------------------------------------------------------------------------------- autograd
@pytest.mark.parametrize("interleaved", [False, True])
def test_autograd_rope(interleaved):
    """A model that calls it: logits = rope(x W) read out, cross-entropy; the gradient of W against 64-bit differences of the
    formula, and a shared leaf's gradients summed."""
    from zillaphp_b200 import autograd as ag
    g = np.random.default_rng(41)
    rows, heads, dim, rot = 6, 2, 8, 6
    x0, w0, u0 = g.standard_normal((rows, 5)), g.standard_normal((5, heads * dim)) * 0.4, g.standard_normal((heads * dim, 7)) * 0.4
    pos, y = np.array([0, 1, 5, 70, 4000, -3]), np.array([0, 6, 3, 2, 1, 5])
    plan = R.rates(rot, 10000.0, 3, 4.0, 64)

    def loss64(w):
        z = torch.from_numpy(x0 @ w).reshape(rows, heads, dim)
        z, _ = R.rotate(z, torch.from_numpy(pos), rot, int(interleaved), plan)
        z = z.reshape(rows, -1) @ torch.from_numpy(u0)
        return float(torch.nn.functional.cross_entropy(z, torch.from_numpy(y)))

    table = ag.RopeTable(rot, scaling="parts", factor=4.0, original=64)
    w, u = ag.Parameter(w0), ag.Parameter(u0)
    x = ag.Tensor.from_numpy(x0)

    def forward():
        z = x.matmul(w)
        h = z.view((rows, heads, dim))
        h._attach((z,), "view", lambda g_: z.accumulate_grad(g_.view(z.shape)))
        r = h.rope(pos, table, interleaved)
        flat = r.view((rows, heads * dim))
        flat._attach((r,), "view", lambda g_: r.accumulate_grad(g_.view(r.shape)))
        return ag.CrossEntropy()(flat.matmul(u), y)

    loss = forward()
    w64 = w.numpy().astype(np.float64)
    assert abs(loss.item() - loss64(w64)) < 1e-5
    loss.backward()
    grad = w.grad.numpy().astype(np.float64)
    # central differences in 64 bits: step 1e-4, their own error below step^2 times a third derivative of order 1; fp32: sums
    # of a few dozen products of order 1, 2^-24 each
    for i in range(5):
        for j in range(heads * dim):
            e = np.zeros_like(w64)
            e[i, j] = 1e-4
            d = (loss64(w64 + e) - loss64(w64 - e)) / 2e-4
            assert abs(d - grad[i, j]) < 1e-5, (i, j, d, grad[i, j])
    w.grad = None
    a, b = forward(), forward()
    a.backward()
    b.backward()
    assert np.max(np.abs(w.grad.numpy() - 2 * grad)) < 1e-5
    with ag.no_grad():
        z = ag.Tensor.from_numpy(np.ones((2, 1, 8))).rope([1, 2], table)
        assert not z.requires_grad
    for bad in ([1], [1.0, 2.0], [1, 2 ** 31]):
        with pytest.raises(ValueError):
            ag.Tensor.from_numpy(np.ones((2, 1, 8))).rope(bad, table)


@pytest.mark.parametrize("prefix,length,bound", [(0, 2 ** 31 - 5000, 0), (2 ** 31 - 5000, 1, 1), (1000, 70, 2 ** 31 - 6000)])
def test_attend_lengths_near_31_bits(bufs, prefix, length, bound):
    """Lengths and bounds of lengths whose last slot's end passes 31 bits.  All keys are zero, so that every key weighs the same; the
    tokens' pages are page 0, whose values are 0, but for the last 2^23 keys, whose values are 1."""
    page, T, keys = 128, torch.bfloat16, prefix + length
    kv = PagedKv(2, page, 1, 32, "bf16")
    bufs.write(kv.v_id, torch.stack([torch.zeros(1, page, 32), torch.ones(1, page, 32)]).to(T))
    ones = min(1 << 23, (keys - 1) // page * page // 2) // page * page      # whole pages at the end, a part of one more
    table = torch.zeros(-(-max(length, bound) // page), dtype=torch.int32)
    front = torch.zeros(max(1, -(-prefix // page)), dtype=torch.int32)
    long_, n = (front, prefix) if prefix > length else (table, length)
    last = -(-n // page)
    long_[last - ones // page: last] = 1
    light = n - (last * page - ones)                                          # keys of value 1
    q, io = torch.ones((1, 1, 32)).to(T), bufs.put(torch.full((1, 1, 32), 7.0).to(T))
    work = kv.attend_work(1, 1, 1, prefix, 1, bound or length)
    kv.attend(bufs.put(q), io, bufs.put(i32([0, 1])), bufs.put(i32([length])), bufs.put(table), bufs.put(front), 1, 1, 1, table.numel(), prefix, 1,
              bound or length, 1.0, bufs.new(max(1, work)))
    got, want = bufs.get(io, (1, 1, 32), T).double(), light / keys
    # counts up to 2^24 are exact in fp32; the joined sums round at most 2^-24 a slot (under 2000), the result once
    assert ((got - want).abs() <= want * (2.0 ** -8 + 2000 * 2.0 ** -24)).all(), (got[0, 0, 0], want)
    kv.close()


def run_attend_minus_infinity(bufs, dtype, new, length, hq, hk, dim, page, prefix, front_gone, own_gone):
    """The first front_gone keys of the prefix and the first own_gone of each sequence (whole pages) score -inf for every
    row; the others score about -100, far below any starting value.  The reference leaves those keys out."""
    T = R.DT[dtype]
    start, pages, front, count, most = batch_of(new, length, prefix, page, 51)
    g = torch.Generator().manual_seed(52)
    k, v = (torch.randn((count, hk, page, dim), generator=g).to(T) for _ in range(2))
    q = torch.randn((start[-1], hq, dim), generator=g).to(T)
    scale = 1 / math.sqrt(dim)
    q[..., 0] = 1.0
    q[..., 1] = 8.0
    k[..., 1] = -100.0 / (8.0 * scale)
    gone = torch.cat([front[: front_gone // page]] + [r[: own_gone // page] for r in pages]).long()
    seen = k.clone()
    seen[gone, :, :, 0] = -math.inf
    kv = PagedKv(count, page, hk, dim, dtype)
    bufs.write(kv.k_id, seen)
    bufs.write(kv.v_id, v)
    io = bufs.put(torch.full((start[-1], hq, dim), 7.0).to(T))
    work = kv.attend_work(len(new), start[-1], hq, prefix, max(new), max(length))
    kv.attend(bufs.put(q), io, bufs.put(i32(start)), bufs.put(i32(length)), bufs.put(pages), bufs.put(front), len(new), start[-1], hq, most, prefix,
              max(new), max(length), scale, bufs.new(max(1, work)))
    got = bufs.get(io, (start[-1], hq, dim), T)
    ref = R.attend(q, k, v, start, [n - own_gone for n in length], [r[own_gone // page:] for r in pages.tolist()],
                   front[front_gone // page:].tolist(), prefix - front_gone, scale, page)
    err = (got.double() - ref[0]).abs()
    tol = R.attend_tolerance(ref, dim, T)
    assert (err <= tol).all(), float((err / tol).nan_to_num(math.inf).max())
    kv.close()


@pytest.mark.parametrize("dtype,new,length,hq,hk,dim,page,prefix,front_gone,own_gone", [
    ("bf16", [1] * 33, [9] * 33, 32, 8, 128, 64, 1000, 64, 0),       # the prefix on tcgen05: a step, a tile, all of a block's tiles
    ("fp16", [1] * 33, [9] * 33, 32, 8, 128, 64, 1000, 128, 0),
    ("bf16", [3] * 11, [40] * 11, 32, 4, 64, 16, 3000, 1600, 0),
    ("fp16", [2] * 40, [3] * 40, 16, 8, 32, 16, 4000, 208, 0),
    ("bf16", [4] * 30, [30] * 30, 16, 2, 128, 128, 2000, 1920, 0),
    ("bf16", [1] * 33, [9] * 33, 32, 8, 128, 64, 1024, 1024, 0),     # nothing is left of the prefix
    ("bf16", [2, 1], [300, 290], 4, 2, 64, 16, 400, 256, 128),        # the other kernels
    ("fp16", [5, 30], [300, 290], 8, 1, 64, 32, 400, 64, 64),
    ("bf16", [1, 2], [80, 90], 4, 2, 64, 16, 96, 64, 32),             # in one launch
])
def test_attend_keys_that_score_minus_infinity(bufs, dtype, new, length, hq, hk, dim, page, prefix, front_gone, own_gone):
    run_attend_minus_infinity(bufs, dtype, new, length, hq, hk, dim, page, prefix, front_gone, own_gone)


def border_row(g, vocab, side, with_q):
    """A row p, q and a number u whose border is known exactly: one large weight and the rest near 2^-27, in multiples of 2^-62,
    some weights behind token t (which comes soon after the large one) moved until the sum up to t is 2^-40 of the whole sum above (side 1) u times that, or below it
    (side -1).  Returns p, q, u and the token that has to be drawn."""
    p = g.integers((1 << 23) + (1 << 20), (1 << 24) - (1 << 20), vocab).astype(np.int64)      # units of 2^-50: 2^-27 to 2^-26
    q = g.integers(0, 1 << 20, vocab).astype(np.int64) if with_q else np.zeros(vocab, np.int64)   # units of 2^-62
    h = int(g.integers(0, vocab * 3 // 4))
    p[h] = 3 << 48                                                         # 0.75
    p[vocab - 1] = q[vocab - 1] = 0                                        # the draft that fails
    c = np.cumsum((p << 12) - q)
    big = 1 << 24
    u = -(-int(c[h + 20]) * big // int(c[-1]))                             # a few tokens behind the large one
    t = int(np.searchsorted(c.astype(np.float64), u / big * float(c[-1])))
    d = int(c[t]) * big - u * int(c[-1]) - side * (int(c[-1]) >> 16)       # what the border is too high by, times 2^24
    more = d // u >> 12                                                    # units of 2^-50 behind t
    each, rest = divmod(abs(more), 64)
    sign = 1 if more > 0 else -1
    p[t + 1: t + 65] += sign * each
    p[t + 1] += sign * rest
    c = np.cumsum((p << 12) - q)
    d = int(c[t]) * big - u * int(c[-1])
    assert int(c[-1]) >> 17 < side * d < int(c[-1]) >> 15 and h < t and t + 65 < vocab and p[t + 1: t + 65].min() >= 1 << 23 and p[t + 1: t + 65].max() < 1 << 24
    return (p * 2.0 ** -50).astype(np.float32), (q * 2.0 ** -62).astype(np.float32), np.float32(u / big), t if side > 0 else t + 1


@pytest.mark.parametrize("with_q", [False, True])
@pytest.mark.parametrize("vocab,ld,batch", [(1 << 22, 1 << 22, 4), (3_000_001, 3_000_001, 6), (300_000, 300_000, 8), (300_001, 300_001, 40), (300_001, 300_004, 40)])
def test_verify_next_to_a_border(bufs, vocab, ld, batch, with_q):
    """One large weight and many small ones: each sum has to be good to 2^-42, so that a border 2^-40 away is on its side."""
    g = np.random.default_rng(vocab + batch)
    n = 2 if with_q else 1
    p, q, u, want = np.zeros((n * batch, ld), np.float32), np.zeros((n * batch, ld), np.float32), np.zeros(n * batch, np.float32), []
    for b in range(batch):
        p[n * b, :vocab], q[n * b, :vocab], u[n * b + n - 1], token = border_row(g, vocab, 1 if b % 2 else -1, with_q)
        want += [token, -1][:n]
    draft = np.full(n * batch, vocab - 1, np.int32)
    it, ia = bufs.new(n * batch), bufs.new(batch)
    ip, iq = bufs.put(torch.from_numpy(p)), bufs.put(torch.from_numpy(q)) if with_q else 0
    bufs.be.draftVerifyDev(ip, ld, iq, ld, bufs.put(torch.from_numpy(draft)), bufs.put(torch.from_numpy(u)), bufs.put(i32(range(0, n * batch + 1, n))), it, ia,
                           batch, n * batch, vocab)
    assert bufs.get(it, (n * batch,), torch.int32).tolist() == want
    assert bufs.get(ia, (batch,), torch.int32).tolist() == [0] * batch


@pytest.mark.parametrize("vocab,ld", [(700, 700), (701, 701), (100_003, 100_004), (100_003, 100_003)])
@pytest.mark.parametrize("batch", [1, 160])
def test_verify_largest_weights(bufs, vocab, ld, batch):
    """Infinite weights count as the largest finite number; several of those in one thread's elements, alone and as residuals."""
    top, inf, g = np.finfo(np.float32).max, np.float32(np.inf), np.random.default_rng(71)
    p, q = np.zeros((3 * batch, ld), np.float32), np.zeros((3 * batch, ld), np.float32)
    p[:, :vocab] = g.random((3 * batch, vocab), np.float32)
    q[:, :vocab] = g.random((3 * batch, vocab), np.float32)
    u, draft, new = g.random(3 * batch).astype(np.float32), np.full(3 * batch, 3, np.int32), [2, 1] * batch
    p[0::3, 3] = 0.0                                                         # the draft fails: residuals
    p[:, [4, 5, 6, 7, 36, 37, 68, 132, 133, 260]] = top
    p[:, [5, 37, 640]] = inf
    p[:, 641] = top / 1000                                                   # finite weights keep their proportions
    q[:, [36, 68]] = top                                                     # no residual there
    q[:, 132] = -top                                                         # twice the largest number
    q[:, 6] = inf
    finite = np.minimum(p, top)
    start = starts(new)
    it, ia = bufs.new(3 * batch), bufs.new(2 * batch)
    bufs.be.draftVerifyDev(bufs.put(torch.from_numpy(p)), ld, bufs.put(torch.from_numpy(q)), ld, bufs.put(torch.from_numpy(draft)),
                           bufs.put(torch.from_numpy(u)), bufs.put(i32(start)), it, ia, 2 * batch, 3 * batch, vocab)
    tokens, accepted = R.verify(finite, q, draft, u, start, vocab)
    assert bufs.get(it, (3 * batch,), torch.int32).tolist() == [tokens[i] for i in range(3 * batch)]
    assert bufs.get(ia, (2 * batch,), torch.int32).tolist() == accepted


@pytest.mark.parametrize("hq,hk,dim,prefix,new", [(4, 2, 64, 300, [1, 1, 2]), (4, 2, 64, 100, [1, 1, 2]), (64, 2, 128, 3000, [2, 1, 2]), (96, 1, 64, 4100, [1, 1, 1])])
def test_attend_no_own_keys_at_all(bufs, hq, hk, dim, prefix, new):
    """max_len 0: every row sees the prefix alone, and a sequence with a length all the same is recorded and left as it is."""
    lib, page, T = native.load(), 16, torch.bfloat16
    start, pages, front, count, most = batch_of(new, [0] * 3, prefix, page, 61)
    g = torch.Generator().manual_seed(62)
    k, v = (torch.randn((count, hk, page, dim), generator=g).to(T) for _ in range(2))
    q = torch.randn((start[-1], hq, dim), generator=g).to(T)
    kv = PagedKv(count, page, hk, dim, "bf16")
    bufs.write(kv.k_id, k)
    bufs.write(kv.v_id, v)
    before = torch.full((start[-1], hq, dim), 7.0).to(T)
    iq, it, ip, front_id = bufs.put(q), bufs.put(i32(start)), bufs.put(pages), bufs.put(front)
    work = bufs.new(max(1, kv.attend_work(3, start[-1], hq, prefix, max(new), 0)))
    ref = R.attend(q, k, v, start, [0] * 3, pages.tolist(), front.tolist(), prefix, 0.1, page)
    tol = R.attend_tolerance(ref, dim, T)
    for length in ([0, 0, 0], [0, 5, 0]):
        io = bufs.put(before)
        kv.attend(iq, io, it, bufs.put(i32(length)), ip, front_id, 3, start[-1], hq, most, prefix, max(new), 0, 0.1, work)
        got = bufs.get(io, before.shape, T)
        ok = torch.tensor([length[b] == 0 for b in range(3) for _ in range(new[b])])
        assert ((got.double() - ref[0]).abs() <= tol)[ok].all()
        assert torch.equal(got[~ok], before[~ok])
        assert lib.zilla_check_device() == (-3 if any(length) else 0)
    kv.close()


@pytest.mark.parametrize("spare", [0, 2000])
@pytest.mark.parametrize("start,bad", [
    ([0, 2, 9], [1]), ([0, 2, 4, 6], [2]), ([0, 2, 4, 9, 12], [2, 3]), ([-1, 1, 3], [0]), ([0, 2, 2 ** 31 - 1], [1]), ([-2 ** 31, 2, 4], [0]),
    ([0, 2, 1, 1], [1]), ([0, 3, -5], [1])])
def test_append_rows_that_do_not_fit_are_recorded(bufs, start, bad, spare):
    """A sequence with rows outside the call's four, or with fewer than none, is recorded and none of its rows is stored; the
    others are.  Alone, and in front of many empty sequences; there, a start that steps back may cost the others their rows too
    (which are found between starts that rise), but stores nothing wrong."""
    lib, T = native.load(), torch.bfloat16
    size, rows = len(start) - 1, 4
    kv = PagedKv(size + 1, 16, 1, 32, "bf16")
    shape = (size + 1, 1, 16, 32)
    want_k = torch.full(shape, 3.0).to(T)
    bufs.write(kv.k_id, want_k)
    bufs.write(kv.v_id, want_k)
    x, want = torch.arange(1, rows + 1).float()[:, None].expand(rows, 32).contiguous(), torch.full((rows, 1, 32), 7.0).to(T)
    ix, io, total = bufs.put(x), bufs.put(want), size + spare
    kv.append(0, ix, 0, 32, ix, 0, 32, ix, 0, 32, io, bufs.put(i32(start + [start[-1]] * spare)), bufs.put(i32([16] * total)),
              bufs.put(i32([[min(b, size)] for b in range(total)])), total, rows, 1, 1, 0, 0, 0)
    for b in range(size):
        for t in range(start[b], start[b + 1]) if b not in bad else ():
            want[t] = x[t].to(T)
            want_k[b, :, 16 - start[b + 1] + t] = x[t].to(T)
    assert lib.zilla_check_device() == -3 and lib.zilla_check_device() == 0
    got, got_k, got_v = bufs.get(io, want.shape, T), bufs.get(kv.k_id, shape, T), bufs.get(kv.v_id, shape, T)
    if spare and any(start[b] > start[b + 1] for b in range(size)):
        want, want_k = torch.where(got == 7.0, got, want), torch.where(got_k == 3.0, got_k, want_k)
    assert torch.equal(got, want) and torch.equal(got_k, want_k) and torch.equal(got_v, want_k)
    kv.close()


@pytest.mark.parametrize("dtype,dim,hq,hk,page,prefix,new,length", [
    ("bf16", 128, 8, 2, 64, 0, [300, 1, 513], [300, 40, 700]),          # prompts from their first token, and behind earlier ones
    ("fp16", 64, 16, 2, 16, 100, [257, 64, 0, 130], [257, 64, 9, 1000]),
    ("bf16", 128, 8, 1, 64, 1500, [400, 129], [400, 500]),              # the prefix on tcgen05
    ("fp16", 32, 4, 4, 128, 2500, [1, 650], [300, 651]),
    ("bf16", 64, 2, 2, 32, 3, [190] * 3, [190, 1, 200]),                # more new rows than keys
])
def test_attend_prompts(bufs, dtype, dim, hq, hk, page, prefix, new, length):
    """Hundreds of new rows a sequence, as a prompt's pass has them."""
    run_attend(bufs, dtype, new, length, hq, hk, dim, page, prefix, 2)


@pytest.mark.parametrize("dtype,hq,dim,rot,interleaved", [("bf16", 6, 64, 64, 0), ("fp16", 3, 128, 40, 1), ("bf16", 5, 32, 30, 0)])
def test_append_in_place(bufs, dtype, hq, dim, rot, interleaved):
    """The queries rotated where they lie, for rows of the cache's type without gaps."""
    T, new = R.DT[dtype], [40, 0, 3]
    start, pages, _, count, most = batch_of(new, [50, 7, 3], 0, 16, 81)
    g = torch.Generator().manual_seed(82)
    rows = start[-1] + 2
    q, k, v = (torch.randn((rows, h, dim), generator=g).to(T) for h in (hq, 1, 1))
    kv = PagedKv(count, 16, 1, dim, dtype)
    table = bufs.new(rot + 2)
    bufs.be.ropeTableDev(table, rot)
    iq = bufs.put(q)
    kv.append(R.CODE[dtype], iq, 0, hq * dim, bufs.put(k), 0, dim, bufs.put(v), 0, dim, iq, bufs.put(i32(start)), bufs.put(i32([50, 7, 3])), bufs.put(pages),
              3, rows, hq, most, 11, table, rot, interleaved)
    got, pos = bufs.get(iq, q.shape, T), 11 + torch.tensor(list(range(10, 50)) + [0, 1, 2])
    ref, size = R.rotate(q[:-2], pos, rot, interleaved, R.rates(rot))
    assert ((got[:-2].double() - ref).abs() <= size * (R.ROTATION + R.far(pos)) + R.half_step(ref, T)).all()
    assert torch.equal(got[-2:], q[-2:])
    kv.close()


def test_a_buffer_that_took_the_place_of_a_caches(bufs):
    """A cache whose buffer was freed stays refused when a new buffer has the handle and the memory of the old one, and does not
    free that one."""
    be, lib = bufs.be, native.load()
    for which in range(2):
        kv = PagedKv(4, 16, 2, 32, "bf16")
        freed = (kv.k_id, kv.v_id)[which]
        be.bufferFree(freed)
        mine = [be.bufferAlloc(4 * 16 * 2 * 32 // 2) for _ in range(3)]
        assert freed in mine                                    # the first free handle, and as a rule the same memory
        want = torch.arange(4 * 16 * 2 * 32 // 2).float()
        for i in mine:
            bufs.write(i, want)
        assert lib.zilla_kv_k_id(kv.id) == -1 and lib.zilla_kv_v_id(kv.id) == -1
        assert lib.zilla_kv_attend_work(kv.id, 1, 1, 2, 0, 1, 16) == -1
        kv.close()
        for i in mine:
            assert torch.equal(bufs.get(i, want.shape, torch.float32), want)
            be.bufferFree(i)
