"""The 8-bit cache at the ends of its range: sequences that the partition
splits, blocks far into a large cache, scales and values of any size, calls
that run into their wait limit, and what is refused.

Outputs are held to sharp_bound, which knows no scale but those that matter:
a block of negligible weight may not cost another one precision.
"""
import pytest
import torch

from clove_b200 import _lib
from fp8_reference import RefPool
from test_gpu_fp8 import DEV, i32, make_pool, run_decode, tables_for

pytestmark = pytest.mark.gpu

# ---------------------------------------------------------------------------
# sequences that are split between CTAs
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,bs,H,G,D", [(torch.float32, 16, 2, 4, 128), (torch.float32, 64, 1, 2, 256),
                                            (torch.float32, 256, 2, 8, 128), (torch.float16, 8, 2, 3, 64),
                                            (torch.bfloat16, 256, 2, 1, 64), (torch.bfloat16, 32, 2, 8, 256),
                                            (torch.float16, 128, 1, 5, 128), (torch.float32, 8, 1, 7, 64)])
@pytest.mark.parametrize("append,accumulate", [(False, False), (True, False), (False, True), (True, True)])
def test_long_windows(dtype, bs, H, G, D, append, accumulate):
    # windows that start inside a block and a slice, of sequences longer and shorter than them
    for window in (1025, 1777):
        run_decode([3000, 1776, 0, 1777, 5, 4999, 1], bs, H, G, D, dtype, seed=window + bs + G, append=append,
                   window=window, accumulate=accumulate, softcap=15.0 if G == 8 else 0.0, alibi=G % 2 == 1)


@pytest.mark.parametrize("dtype,bs,H,G,D", [(torch.bfloat16, 16, 8, 2, 64), (torch.float32, 32, 6, 1, 128),
                                            (torch.float16, 64, 5, 1, 256), (torch.bfloat16, 256, 8, 4, 64)])
@pytest.mark.parametrize("window", [1, 33, 200, 0])
@pytest.mark.parametrize("append,accumulate", [(False, False), (True, True)])
def test_many_short_windows(dtype, bs, H, G, D, window, append, accumulate):
    # more KV heads than are taken whole: short windows through the partition
    gen = torch.Generator().manual_seed(window + bs)
    lens = torch.randint(0, 300, (125,), generator=gen)
    lens[::11], lens[7], lens[124] = 0, 1000, 513
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    assert lens.numel() * H > 4 * sms
    run_decode(lens.tolist(), bs, H, G, D, dtype, seed=window + G, append=append, window=window, accumulate=accumulate)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("bs,H,G,D", [(8, 2, 8, 128), (16, 3, 5, 64), (32, 2, 3, 256), (64, 2, 8, 256), (128, 1, 7, 128),
                                      (256, 2, 2, 64), (256, 1, 1, 256)])
@pytest.mark.parametrize("append", [False, True])
def test_split_sequences(dtype, bs, H, G, D, append):
    run_decode([0, 1, 33, 257, 2600, 1025], bs, H, G, D, dtype, seed=bs + G + D, append=append)


# ---------------------------------------------------------------------------
# far into a large cache
# ---------------------------------------------------------------------------
def test_blocks_beyond_two_gigabytes():
    # codes of the blocks used lie beyond 2^31 bytes of their plane: what the same blocks give in a small cache
    from clove_b200 import Fp8KVPool
    bs, H, D, B, G = 256, 8, 128, 3, 4
    gen = torch.Generator().manual_seed(3)
    lens = [700, 1500, 256]
    used = 24  # blocks 0 .. 23 of the small cache are the last ones of the large one
    nb = 2 ** 31 // (bs * H * D) + 100
    small, first = make_pool(used, bs, H, D, gen, mass=True), nb - used
    assert first * bs * H * D > 2 ** 31
    big = Fp8KVPool(nb, bs, H, D, track_mass=True)
    big.storage.view(torch.uint8)[:, first:] = small.storage.view(torch.uint8)
    big.scales[:, first:] = small.scales
    big.mass[first:] = small.mass
    ids = torch.randperm(used, generator=gen)
    tables = torch.zeros((B, 7), dtype=torch.int32)
    new = torch.zeros((B, 2), dtype=torch.int32)
    at = 0
    for b, n in enumerate(lens):
        k = n // bs + 1
        tables[b, :k], at = ids[at:at + k], at + k
    new[:] = ids[at:at + 2 * B].reshape(B, 2)
    copies = [int(x) for x in ids[at + 2 * B:at + 2 * B + 2]]
    kv = torch.randn((2, 300, H, D), generator=gen).bfloat16().to(DEV)
    q = torch.randn((B, H * G, D), generator=gen).bfloat16().to(DEV)
    slots = torch.cat([int(tables[1, 2]) * bs + torch.arange(bs), int(tables[0, 0]) * bs + torch.arange(44)])
    got = []
    for pool, off in ((small, 0), (big, first)):
        t, t2 = i32(tables + off), i32(new + off)
        pool.reshape_and_cache(kv[0], kv[1], i32(slots + off * bs))
        outs = [pool.decode(q, t, i32(lens), max_ctx=1501, k_new=kv[0, :B], v_new=kv[1, :B], accumulate=True)]
        outs += pool.gather_kv(t, i32([n + 1 for n in lens]), 1501)
        outs += pool.evict(t, i32([n + 1 for n in lens]), t2, 300, 20, max_ctx=1501)
        pool.copy_blocks(t2[:, 0].contiguous()[:2], i32([c + off for c in copies]))
        outs += [pool.decode(q, t2, outs[-1], max_ctx=300, window=77)]
        assert pool.pool_status() == 0
        outs += [pool.storage.view(torch.uint8)[:, off:], pool.scales[:, off:], pool.mass[off:]]
        got.append(outs)
    for a, b in zip(*got):
        assert torch.equal(a, b)
    assert not big.storage.view(torch.uint8)[:, :first].any()


# ---------------------------------------------------------------------------
# scales of any size
# ---------------------------------------------------------------------------
def sharp_bound(ref, q, tables, lens, scale):
    """(out, bound) in 64 bits for a float32 computation of plain scores.

    Token t's score is a float32 sum of D products, rounded or truncated at
    most D / 16 + 8 times, so off by at most e_t = (D / 16 + 8) 2^-23 S_t, S_t
    its sum of magnitudes; exp2, the two halves of a weight and the sums over L
    tokens add c = (L / 32 + 24) 2^-23.  A weight p_t is thus off by p_t (e_t +
    c) in the numerator, and the denominator by the sum of these.  What a
    weight times its block's scale s_t falls below f16's smallest step is
    rounded at 2^-25 in units in which the largest such product of the row is
    at least 2^10: 2^-35 max(p s) |code_t| for each token."""
    q = q.cpu().double()
    B, hq, D = q.shape
    H = ref.codes.shape[2]
    out, bound = torch.zeros(B, hq, D, dtype=torch.float64), torch.zeros(B, hq, D, dtype=torch.float64)
    for b in range(B):
        L = int(lens[b])
        pos = torch.arange(L)
        k, v = (ref.rows(p, tables[b].cpu(), pos) for p in range(2))
        blk = tables[b].cpu().long()[pos // ref.bs]
        for h in range(H):
            g = slice(h * (hq // H), (h + 1) * (hq // H))
            z = scale * q[b, g] @ k[:, h].t()
            e = (D / 16 + 8) * 2.0 ** -23 * (abs(scale) * q[b, g].abs() @ k[:, h].abs().t()) + (L / 32 + 24) * 2.0 ** -23
            p = torch.softmax(z, 1)
            out[b, g] = p @ v[:, h]
            mag = v[:, h].abs()
            top = (p * ref.scales[1][blk, h]).amax(1)
            bound[b, g] = (p * e) @ mag + (p * e).sum(1, keepdim=True) * (p @ mag) + 1e-37 + \
                2.0 ** -35 * top[:, None] * ref.codes[1][blk, h, pos % ref.bs].abs().sum(0)
    return out, bound


def levels(lens, bs, H, G, D, dtype, seed, size, weight):
    """A pool of sequences whose block j holds values of about 2^size(j) and
    scores of about weight(j) in the log2 domain, and what a decode of it gives."""
    from clove_b200 import Fp8KVPool
    gen = torch.Generator().manual_seed(seed)
    tables, nb = tables_for(lens, bs, gen)
    pool = Fp8KVPool(nb, bs, H, D)
    for b, n in enumerate(lens):
        t = torch.arange(n)
        blocks = [int(x) for x in t // bs]
        k, v = torch.randn((n, H, D), generator=gen) * 0.05, torch.randn((n, H, D), generator=gen)
        k[:, :, 0] = torch.tensor([float(weight(j)) for j in blocks])[:, None]
        v *= torch.tensor([2.0 ** size(j) for j in blocks])[:, None, None]
        slots = tables[b].cpu().long()[t // bs] * bs + t % bs
        pool.reshape_and_cache(k.to(DEV), v.to(DEV), i32(slots))
    ref = RefPool(pool.storage, pool.scales)
    q = (torch.randn((len(lens), H * G, D), generator=gen) * 0.5).to(dtype)
    q[:, :, 0] = 1.0
    scale = 0.6931471805599453  # scores in the log2 domain
    want, bound = sharp_bound(ref, q, tables, lens, scale)
    out = pool.decode(q.to(DEV), tables, i32(lens), scale=scale, max_ctx=max(lens))
    assert pool.pool_status() == 0
    err = (out.cpu().double() - want).abs()
    assert (err <= bound).all(), f"{float((err / bound).max()):.3g} of the bound"


SHAPES = [(torch.bfloat16, 16, 2, 4, 128), (torch.float16, 8, 2, 8, 64), (torch.float32, 32, 1, 1, 256),
          (torch.float32, 64, 1, 8, 128), (torch.bfloat16, 256, 1, 2, 64), (torch.float16, 128, 1, 6, 256)]


@pytest.mark.parametrize("dtype,bs,H,G,D", SHAPES)
@pytest.mark.parametrize("ratio", [3, 6, 26, 40, 100])
@pytest.mark.parametrize("at", ["first", "middle", "last"])
def test_a_loud_block_of_no_weight(dtype, bs, H, G, D, ratio, at):
    # one block's values are 2^ratio times the others', its tokens weigh nothing
    for lens in ([3 * bs + 5, 700], [9 * bs + 1, 6000]):
        for n in lens:
            last = (n - 1) // bs
            j0 = {"first": 0, "middle": (last + 1) // 2, "last": last}[at]
            levels([n], bs, H, G, D, dtype, ratio + n, lambda j: ratio if j == j0 else 0, lambda j: -220 if j == j0 else 0)


@pytest.mark.parametrize("dtype,bs,H,G,D", SHAPES)
@pytest.mark.parametrize("ratio", [6, 26, 60, 100])
def test_loud_blocks_of_little_weight(dtype, bs, H, G, D, ratio):
    # every other block's values are 2^ratio times the others', its tokens' weights as much smaller: they count alike
    levels([700, 9 * bs + 1], bs, H, G, D, dtype, ratio, lambda j: ratio * (j & 1), lambda j: -ratio * (j & 1))
    levels([4000], bs, H, G, D, dtype, ratio, lambda j: -ratio * (j & 1), lambda j: ratio * (j & 1))


@pytest.mark.parametrize("dtype,bs,H,G,D", SHAPES)
@pytest.mark.parametrize("slope", [-2.0, -1.0, -0.5, 0.0, 1.0])
@pytest.mark.parametrize("way", [1, -1])
def test_scales_in_steps(dtype, bs, H, G, D, slope, way):
    # values grow or shrink from block to block over 2^120, weights with slope times that
    n = 24 * bs - 3
    levels([n], bs, H, G, D, dtype, 5, lambda j: way * (5 * j - 60), lambda j: slope * way * (5 * j - 60))


@pytest.mark.parametrize("dtype,bs,H,G,D", SHAPES)
@pytest.mark.parametrize("power", [-20, 0, 30, 110])
@pytest.mark.parametrize("tilt", [-60, 0, 25])
def test_blocks_of_zeros(dtype, bs, H, G, D, power, tilt):
    # blocks whose values are all 0 have the smallest scale there is, 2^-126, and any weight: in front and in between
    for n, zeros in ((700, lambda j: j < 2), (9 * bs + 1, lambda j: j % 3 == 0), (3000, lambda j: j < 5 or j % 4 == 2)):
        levels([n], bs, H, G, D, dtype, 7, lambda j: -400 if zeros(j) else power, lambda j: tilt if zeros(j) else 0)


@pytest.mark.parametrize("dtype,bs,H,G,D", SHAPES)
def test_scales_of_each_kv_head_and_query_apart(dtype, bs, H, G, D):
    # random sizes and weights, independent of one another
    gen = torch.Generator().manual_seed(1)
    size = torch.randint(-50, 50, (800,), generator=gen).tolist()
    weight = (torch.randn((800,), generator=gen) * 40).tolist()
    levels([900, 5000, 17], bs, H, G, D, dtype, 6, lambda j: size[j], lambda j: weight[j])


# ---------------------------------------------------------------------------
# values near the end of float32
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,bs,H,G,D", SHAPES)
@pytest.mark.parametrize("power", [100, 116, 120])
def test_large_values(dtype, bs, H, G, D, power):
    # the values' sums before the division by the weights' stay finite
    levels([700, 2600], bs, H, G, D, dtype, power, lambda j: power, lambda j: 0)


@pytest.mark.parametrize("dtype,G,D", [(torch.bfloat16, 4, 128), (torch.float32, 8, 64), (torch.float16, 1, 256)])
@pytest.mark.parametrize("exponent", [-149, -127, 125, 126, 127])
def test_scales_at_the_ends_of_float32(dtype, G, D, exponent):
    # any positive finite scale: a loaded cache's may be the smallest and the largest
    gen = torch.Generator().manual_seed(8)
    lens = [100, 1300]
    tables, nb = tables_for(lens, 16, gen)
    pool = make_pool(nb, 16, 1, D, gen, scales=(-8, -5))
    pool.storage.view(torch.uint8)[1] &= 0x9F  # values below 2^-2
    pool.scales[1] = 2.0 ** exponent
    ref = RefPool(pool.storage, pool.scales)
    q = torch.randn((2, G, D), generator=gen).to(dtype)
    want, bound = sharp_bound(ref, q, tables, lens, 0.1)
    out = pool.decode(q.to(DEV), tables, i32(lens), scale=0.1, max_ctx=1300)
    assert ((out.cpu().double() - want).abs() <= bound).all()


@pytest.mark.parametrize("G,D", [(4, 128), (8, 64), (1, 256)])
def test_queries_near_the_end_of_float32(G, D):
    gen = torch.Generator().manual_seed(9)
    lens = [100, 1300]
    tables, nb = tables_for(lens, 16, gen)
    pool = make_pool(nb, 16, 1, D, gen, scales=(-8, -5))
    ref = RefPool(pool.storage, pool.scales)
    q = torch.randn((2, G, D), generator=gen) * 2.0 ** 120
    q[:, :, 3], q[:, :, 5] = torch.finfo(torch.float32).max, -torch.finfo(torch.float32).max
    scale = 2.0 ** -126
    want, bound = sharp_bound(ref, q, tables, lens, scale)
    out = pool.decode(q.to(DEV), tables, i32(lens), scale=scale, max_ctx=1300)
    assert ((out.cpu().double() - want).abs() <= bound).all()


# ---------------------------------------------------------------------------
# calls that run into their wait limit
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("append", [False, True])
@pytest.mark.parametrize("bs,lens", [(16, [600, 40]), (16, [5000, 900]), (256, [5000, 900])], ids=["whole", "split", "slices"])
def test_stuck_wait_adds_no_weights(bs, lens, append):
    # the test hook leaves one stage unfilled: the call ends, says so, and leaves the weights as they were, but for
    # that of the token it appends; the next call is right
    gen = torch.Generator().manual_seed(57)
    tables, nb = tables_for([n + 1 for n in lens], bs, gen)
    pool = make_pool(nb, bs, 2, 128, gen, mass=True, scales=(-9, -5))
    q = torch.randn((2, 8, 128), generator=gen)
    kv = torch.randn((2, 2, 2, 128), generator=gen)
    kw = dict(max_ctx=max(lens) + 1, accumulate=True)
    if append:
        kw |= dict(k_new=kv[0].to(DEV), v_new=kv[1].to(DEV))
    before = pool.mass.clone()
    torch.full((1 << 26,), float("nan"), device=DEV)  # what the allocator gives as scratch next
    L = _lib.lib()
    torch.cuda.synchronize()
    try:
        _lib.check(L.clove_cuda_debug_set(2000, 1))
        pool.decode(q.to(DEV), tables, i32(lens), **kw)
        assert pool.pool_status() & _lib.FLAG_TIMEOUT
    finally:
        L.clove_cuda_debug_set(0, 0)
    if append:
        for b, n in enumerate(lens):
            before[int(tables[b, n // bs]), :, n % bs] = pool.mass[int(tables[b, n // bs]), :, n % bs]
    assert torch.equal(pool.mass, before)
    pool.reshape_and_cache(kv[0].to(DEV), kv[1].to(DEV), i32([int(tables[b, n // bs]) * bs + n % bs for b, n in enumerate(lens)]))
    ref = RefPool(pool.storage, pool.scales, pool.mass)
    if append:
        ref.append(kv[0], kv[1], torch.tensor([int(tables[b, n // bs]) * bs + n % bs for b, n in enumerate(lens)]))
    want, bound = ref.decode(q, tables, [n + append for n in lens], 128 ** -0.5, accumulate=True)
    out = pool.decode(q.to(DEV), tables, i32(lens), **kw)
    assert pool.pool_status() == 0
    assert ((out.cpu().double() - want).abs() <= bound).all()
    assert ((pool.mass.cpu().double() - ref.mass).abs() <= ref.mass_bound).all()


# ---------------------------------------------------------------------------
# check flags
# ---------------------------------------------------------------------------
def test_no_flag_is_lost_to_a_read_on_another_stream():
    # flags raised on one stream at any time while another one's reads are under way: each is reported
    gen = torch.Generator().manual_seed(10)
    pool = make_pool(4, 16, 2, 64, gen)
    kv = torch.randn((2, 1, 2, 64), generator=gen).to(DEV)
    bad, side = i32([64]), torch.cuda.Stream()
    torch.cuda.synchronize()
    for i in range(400):
        with torch.cuda.stream(side):
            torch.cuda._sleep(20000 + 173 * i)
            pool.reshape_and_cache(kv[0], kv[1], bad)
        seen, over = 0, False
        while not over:
            over = side.query()
            seen |= pool.pool_status()
        assert seen == _lib.FLAG_SLOT_OOB, i
    assert pool.pool_status() == 0


# ---------------------------------------------------------------------------
# arguments
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("softcap", [1e-39, 1e-45, 1e-60, 5e-324])
def test_caps_too_small_for_float32_are_refused(softcap):
    # not rounded to 0, which stands for no cap
    pool = make_pool(4, 16, 2, 64, torch.Generator().manual_seed(11))
    with pytest.raises((ValueError, _lib.CloveError)):
        pool.decode(torch.ones((1, 4, 64), device=DEV), i32([[0, 1]]), i32([20]), max_ctx=20, softcap=softcap)
    assert pool.pool_status() == 0


@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31, 2 ** 32, 2 ** 32 + 5, 2 ** 63 - 1])
def test_windows_longer_than_any_sequence(window):
    pool = make_pool(4, 16, 2, 64, torch.Generator().manual_seed(12), scales=(-9, -6))
    args = (torch.ones((1, 4, 64), device=DEV), i32([[0, 1]]), i32([20]))
    assert torch.equal(pool.decode(*args, max_ctx=20, window=window), pool.decode(*args, max_ctx=20))


def test_integers_beyond_32_bits_are_refused():
    # not wrapped around to small ones
    pool = make_pool(4, 16, 2, 64, torch.Generator().manual_seed(12), mass=True, scales=(-9, -6))
    bt, cl, q = i32([[0, 1]]), i32([20]), torch.ones((1, 4, 64), device=DEV)
    for n in (2 ** 31, 2 ** 32 + 20, -2 ** 32 + 20):
        for bad in (lambda: pool.decode(q, bt, cl, max_ctx=n), lambda: pool.gather_kv(bt, cl, n),
                    lambda: pool.evict(bt, cl, i32([[2]]), 16, max_ctx=n), lambda: pool.evict(bt, cl, i32([[2]]), n, max_ctx=20),
                    lambda: pool.decode(q, bt, cl, max_ctx=20, window=-abs(n))):
            with pytest.raises((ValueError, _lib.CloveError)):
                bad()
    assert pool.pool_status() == 0


@pytest.mark.parametrize("budget,max_ctx", [(2 ** 31 - 1, 20), (2 ** 31 - 2 ** 16, 20), (16, 2 ** 31 - 1)])
def test_evictions_larger_than_its_indices_count_are_refused(budget, max_ctx):
    # refused before anything is launched: the buffers are small
    pool = make_pool(4, 256, 2, 64, torch.Generator().manual_seed(13), mass=True)
    bt, new = torch.zeros((1, 2 ** 23), dtype=torch.int32, device=DEV), i32([[2]])
    kept, lens = torch.zeros(64, dtype=torch.int32, device=DEV), i32([20])
    rc = pool._lib.clove_fp8_evict(pool.handle, bt.data_ptr(), bt.shape[1], lens.data_ptr(), 1, max_ctx, new.data_ptr(), 1,
                                   budget, 0, kept.data_ptr(), lens.data_ptr(), None, 0, None)
    assert rc in (_lib.ERR_INVALID_ARG, _lib.ERR_UNSUPPORTED)
    assert pool.pool_status() == 0 and not kept.any()
