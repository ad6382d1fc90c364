"""The 8-bit cache on the GPU against its definitions in 64 bits
(fp8_reference.py).

What is written (codes, scales, kept tokens, moved rows) is compared exactly.
Decode outputs and accumulated weights are held to the bound the reference
derives from the scores' size (see RefPool.decode).  Places that must not be
read hold NaN: rows behind a sequence, rows before a window, other blocks.
"""
import ctypes as C

import pytest
import torch

from clove_b200 import _lib
from fp8_reference import RefPool

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)
F8 = torch.float8_e4m3fn
NAN_CODE = 0x7F


def i32(x):
    return torch.as_tensor(x, dtype=torch.int32).to(DEV)


def tables_for(lens, bs, gen, spare=3, width=None):
    """Disjoint random block tables for the lengths; unused entries -1."""
    need = [(int(n) + bs - 1) // bs for n in lens]
    ids = torch.randperm(sum(need) + spare, generator=gen)[: sum(need)]
    t = torch.full((len(need), width or max(1, max(need))), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        t[b, :n] = ids[at:at + n]
        at += n
    return t.to(DEV), sum(need) + spare


def make_pool(nb, bs, H, D, gen, mass=False, scales=(-11, 1)):
    from clove_b200 import Fp8KVPool
    codes = torch.randint(0, 256, (2, nb, H, bs, D), generator=gen, dtype=torch.uint8)
    codes[(codes & 0x7F) == NAN_CODE] = 0x30
    sc = torch.exp2(torch.randint(scales[0], scales[1], (2, nb, H), generator=gen).float())
    m = (torch.rand((nb, H, bs), generator=gen) if mass else None)
    return Fp8KVPool(nb, bs, H, D, 0, storage=codes.to(DEV).view(F8), scales=sc.to(DEV),
                     mass=None if m is None else m.to(DEV))


def poison(pool, tables, lens, first=None):
    """NaN codes in every row that no sequence's tokens first[b] .. lens[b]-1
    hold, NaN scales in blocks without tokens (a block that holds some, even
    in front of a window, has a scale that an append goes on from)."""
    nb, bs = pool.num_blocks, pool.block_size
    used, scaled = torch.zeros((nb, bs), dtype=torch.bool), torch.zeros(nb, dtype=torch.bool)
    for b, n in enumerate(lens):
        scaled[tables[b, : (int(n) + bs - 1) // bs].cpu().long()] = True
        for t in range(first[b] if first else 0, int(n)):
            used[int(tables[b, t // bs]), t % bs] = True
    raw = pool.storage.view(torch.uint8)
    raw.permute(1, 3, 0, 2, 4)[~used.to(DEV)] = NAN_CODE
    pool.scales[:, ~scaled.to(DEV)] = float("nan")


def same(a, b):
    """Equal, NaN to NaN."""
    a, b = a.detach().float().cpu().double(), b.double()
    return bool(((a == b) | (a.isnan() & b.isnan())).all())


def check_state(pool, ref):
    assert same(pool.storage, ref.codes), "codes"
    assert same(pool.scales, ref.scales), "scales"


# ---------------------------------------------------------------------------
# append
# ---------------------------------------------------------------------------
def run_append(dtype, bs, H, D, slots, nb, seed, special=False, mass=True):
    gen = torch.Generator().manual_seed(seed)
    pool = make_pool(nb, bs, H, D, gen, mass=mass)
    ref = RefPool(pool.storage, pool.scales, pool.mass)
    n = len(slots)
    size = torch.exp2(torch.randint(-9, 6, (2, n, H, 1), generator=gen).float())  # some rows raise a scale, some do not
    kv = (torch.randn((2, n, H, D), generator=gen) * size).to(dtype)
    if special and n:
        kv[0, 0, 0, 0], kv[0, -1, -1, 3], kv[1, 0, 0, 1] = float("inf"), float("-inf"), float("nan")
        kv[1, n // 2] = 0.0
    slots = i32(slots)
    pool.reshape_and_cache(kv[0].to(DEV), kv[1].to(DEV), slots)
    ref.append(kv[0], kv[1], slots)
    check_state(pool, ref)
    if mass:
        assert same(pool.mass, ref.mass)
    return pool


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("bs,H,D", [(8, 3, 64), (16, 8, 128), (32, 2, 256), (64, 1, 128), (256, 2, 64), (256, 1, 256)])
def test_append_prompt(dtype, bs, H, D):
    # from the middle of a block on, over whole blocks, ending inside one; padding among them
    nb = 5
    start = bs // 2 + 1
    slots = list(range(start, min(3 * bs + bs // 2, start + 600))) + [-1, -7] + [4 * bs]
    run_append(dtype, bs, H, D, slots, nb, seed=bs + D)


@pytest.mark.parametrize("bs,D", [(16, 128), (8, 64), (128, 256)])
def test_append_any_order_and_twice_the_same_slot(bs, D):
    gen = torch.Generator().manual_seed(3)
    nb = 6
    slots = torch.randint(-2, nb * bs, (3 * bs,), generator=gen).tolist()  # duplicates: the later token counts
    run_append(torch.bfloat16, bs, 2, D, slots, nb, seed=4)


@pytest.mark.parametrize("n", [1, 2, 33, 128])
def test_append_one_token_each(n):
    gen = torch.Generator().manual_seed(n)
    slots = [16 * b + int(torch.randint(0, 16, (1,), generator=gen)) for b in torch.randperm(n, generator=gen).tolist()]
    run_append(torch.bfloat16, 16, 8, 128, slots, n, seed=n)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_append_infinities_nan_and_zeros(dtype):
    run_append(dtype, 16, 2, 64, list(range(3, 40)), 3, seed=9, special=True)


def test_append_many_tokens():
    # more tokens than a look through slot_mapping per block is meant for
    gen = torch.Generator().manual_seed(12)
    nb, bs = 300, 16
    blocks = torch.randperm(nb, generator=gen)[:260]
    slots = torch.cat([b * bs + torch.arange(bs) for b in blocks])[5:-3]
    pad = torch.full((40,), -1)
    run_append(torch.float16, bs, 1, 64, torch.cat([slots[:1000], pad, slots[1000:]]).tolist(), nb, seed=13)
    mixed = torch.cat([slots, slots[torch.randperm(slots.numel(), generator=gen)[:700]]])
    run_append(torch.float16, bs, 1, 64, mixed[torch.randperm(mixed.numel(), generator=gen)].tolist(), nb, seed=14)


def test_append_again_and_again_keeps_no_trace():
    # the second call's result depends on the cache and its own arguments alone
    gen = torch.Generator().manual_seed(5)
    pool = make_pool(200, 16, 2, 64, gen)
    ref = RefPool(pool.storage, pool.scales)
    for n in (3000, 40, 2100):
        slots = torch.randint(0, 200 * 16, (n,), generator=gen)
        kv = torch.randn((2, n, 2, 64), generator=gen)
        pool.reshape_and_cache(kv[0].to(DEV), kv[1].to(DEV), i32(slots))
        ref.append(kv[0], kv[1], slots)
        check_state(pool, ref)


def test_append_slot_out_of_range_is_flagged_and_skipped():
    gen = torch.Generator().manual_seed(6)
    pool = make_pool(4, 16, 2, 64, gen)
    ref = RefPool(pool.storage, pool.scales)
    kv = torch.randn((2, 3, 2, 64), generator=gen)
    slots = torch.tensor([5, 64, 2 ** 31 - 1])
    pool.reshape_and_cache(kv[0].to(DEV), kv[1].to(DEV), i32(slots))
    ref.append(kv[0], kv[1], slots)
    check_state(pool, ref)
    assert pool.pool_status() == _lib.FLAG_SLOT_OOB
    assert pool.pool_status() == 0


def test_append_takes_strided_rows():
    gen = torch.Generator().manual_seed(7)
    pool = make_pool(4, 16, 2, 64, gen)
    ref = RefPool(pool.storage, pool.scales)
    qkv = torch.randn((20, 3 * 2 * 64), generator=gen)
    k, v = qkv[:, 128:256], qkv[:, 256:]
    d = qkv.to(DEV)
    pool.reshape_and_cache(d[:, 128:256], d[:, 256:], i32(range(20)))
    ref.append(k.reshape(20, 2, 64), v.reshape(20, 2, 64), torch.arange(20))
    check_state(pool, ref)


def test_append_nothing():
    pool = make_pool(2, 16, 2, 64, torch.Generator().manual_seed(8))
    e = torch.empty((0, 2, 64), device=DEV)
    pool.reshape_and_cache(e, e, i32([]))
    assert pool.pool_status() == 0


# ---------------------------------------------------------------------------
# decode
# ---------------------------------------------------------------------------
def run_decode(lens, bs, H, G, D, dtype, seed, append=False, softcap=0.0, alibi=False, window=0, accumulate=False,
               scales=(-11, -5), max_extra=0, scale=None, poisoned=True):
    gen = torch.Generator().manual_seed(seed)
    B, a = len(lens), int(append)
    full = [n + a for n in lens]
    tables, nb = tables_for(full, bs, gen)
    pool = make_pool(nb, bs, H, D, gen, mass=accumulate, scales=scales)
    if poisoned:
        poison(pool, tables, lens, [max(0, f - window) for f in full] if window else None)
    q = torch.randn((B, H * G, D), generator=gen).to(dtype)
    kv = torch.randn((2, B, H, D), generator=gen).to(dtype) * 0.5
    slopes = torch.exp2(-8.0 * torch.arange(1, H * G + 1) / (H * G)) if alibi else None
    ref = RefPool(pool.storage, pool.scales, pool.mass)
    if append:
        slots = torch.tensor([int(tables[b, n // bs]) * bs + n % bs for b, n in enumerate(lens)])
        ref.append(kv[0], kv[1], slots)
    scale = D ** -0.5 if scale is None else scale
    want, bound = ref.decode(q, tables, full, scale, softcap, slopes, window, accumulate)
    new = dict(k_new=kv[0].to(DEV), v_new=kv[1].to(DEV)) if append else {}
    out = torch.full((B, H * G, D), float("nan"), device=DEV)
    pool.decode(q.to(DEV), tables, i32(lens), scale=scale, max_ctx=max(full) + max_extra if max(full) else 0, out=out,
                softcap=softcap, alibi_slopes=None if slopes is None else slopes.to(DEV), window=window,
                accumulate=accumulate, **new)
    assert pool.pool_status() == 0
    err = (out.cpu().double() - want).abs()
    assert (err <= bound).all(), f"{float((err / bound).max()):.3f} of the bound"
    check_state(pool, ref)
    if accumulate:
        off = (pool.mass.cpu().double() - ref.mass).abs()
        assert (off <= ref.mass_bound + 1e-37).all(), f"mass: {float((off / (ref.mass_bound + 1e-37)).max()):.3f} of the bound"
    return pool


LENS = [0, 1, 5, 31, 32, 33, 64, 100, 257, 700]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("bs,H,G,D", [(8, 1, 1, 64), (8, 2, 8, 128), (16, 3, 5, 64), (16, 8, 4, 128), (32, 2, 3, 256),
                                      (64, 2, 8, 256), (128, 1, 7, 128), (256, 2, 2, 64), (256, 1, 1, 256)])
@pytest.mark.parametrize("append", [False, True])
def test_decode(dtype, bs, H, G, D, append):
    run_decode(LENS, bs, H, G, D, dtype, seed=bs + G + D, append=append)


@pytest.mark.parametrize("bs,H,G,D", [(8, 2, 2, 128), (16, 2, 4, 64), (32, 1, 8, 256), (64, 2, 1, 128), (256, 1, 3, 64)])
@pytest.mark.parametrize("kw", [dict(softcap=5.0), dict(alibi=True), dict(window=1), dict(window=30), dict(window=257),
                                dict(window=10 ** 6), dict(softcap=20.0, alibi=True, window=45)],
                         ids=["cap", "alibi", "w1", "w30", "w257", "w1e6", "all"])
@pytest.mark.parametrize("append", [False, True])
def test_decode_scores(bs, H, G, D, kw, append):
    run_decode(LENS, bs, H, G, D, torch.bfloat16, seed=7 + bs, append=append, accumulate=G % 2 == 0, **kw)


@pytest.mark.parametrize("bs,H,G,D", [(8, 2, 3, 64), (16, 8, 4, 128), (32, 2, 8, 128), (64, 1, 1, 256), (256, 2, 5, 128)])
@pytest.mark.parametrize("append", [False, True])
def test_decode_adds_up_weights(bs, H, G, D, append):
    run_decode(LENS, bs, H, G, D, torch.float16, seed=11 + bs, append=append, accumulate=True)


@pytest.mark.parametrize("lens", [[0], [0, 0, 0], [1], [4096], [1, 9000], [3] * 200])
@pytest.mark.parametrize("accumulate", [False, True])
def test_decode_lengths(lens, accumulate):
    run_decode(lens, 16, 2, 4, 128, torch.bfloat16, seed=sum(lens), accumulate=accumulate, poisoned=max(lens) < 5000)


@pytest.mark.parametrize("H,G,append", [(4, 2, True), (5, 8, False)])
def test_decode_large_batch(H, G, append):
    # more sequences than a CTA has threads, empty ones among them
    gen = torch.Generator().manual_seed(61)
    lens = torch.randint(0, 90, (301,), generator=gen)
    lens[::7], lens[128], lens[300] = 0, 1500, 700
    run_decode(lens.tolist(), 16, H, G, 64, torch.bfloat16, seed=62, append=append, accumulate=append)


@pytest.mark.parametrize("softcap", [0.5, 3.0, 10.0, 40.0, 200.0])
@pytest.mark.parametrize("G,D,accumulate", [(4, 128, False), (8, 64, True), (2, 256, True), (1, 128, False)])
def test_decode_cap_from_flat_to_steep(softcap, G, D, accumulate):
    # scores far below the cap, around it and far beyond it: all ranges of the tanh, alone and mixed
    run_decode([300, 1, 70, 1500], 16, 2, G, D, torch.float16, seed=int(10 * softcap) + G, append=True, softcap=softcap,
               alibi=G == 4, accumulate=accumulate)


@pytest.mark.parametrize("D,bs,dtype", [(128, 16, torch.bfloat16), (64, 256, torch.float32), (256, 64, torch.float16)])
@pytest.mark.parametrize("n", [1000, 1024, 1025])
def test_decode_whole_and_split_sequences(D, bs, dtype, n):
    # short sequences are taken whole by a CTA, longer ones split: both sides of the border, with the last block shared
    run_decode([n - 1, 3, 700], bs, 2, 4, D, dtype, seed=n + D, append=True)


@pytest.mark.parametrize("max_extra", [1, 100, 5000])
def test_decode_max_ctx_is_only_a_bound(max_extra):
    gen = torch.Generator().manual_seed(2)
    lens = [5, 300, 0]
    tables, nb = tables_for(lens, 16, gen, width=400)
    pool = make_pool(nb, 16, 2, 64, gen, mass=True)
    ref = RefPool(pool.storage, pool.scales, pool.mass)
    q = torch.randn((3, 4, 64), generator=gen)
    want, bound = ref.decode(q, tables, lens, 0.125, accumulate=True)
    out = pool.decode(q.to(DEV), tables, i32(lens), scale=0.125, max_ctx=300 + max_extra, accumulate=True)
    assert ((out.cpu().double() - want).abs() <= bound).all()
    assert ((pool.mass.cpu().double() - ref.mass).abs() <= ref.mass_bound).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_decode_scales_far_apart(dtype):
    # neighbouring blocks' scales differ by up to 2^40: no block drowns in another's range
    run_decode([40, 700, 333], 16, 2, 4, 128, dtype, seed=21, scales=(-40, 1), scale=0.01)
    run_decode([40, 700, 333], 8, 2, 2, 64, dtype, seed=22, scales=(-30, -20))


@pytest.mark.parametrize("power", [-30, -12, 12])
def test_decode_queries_of_any_size(power):
    gen = torch.Generator().manual_seed(31)
    lens = [3, 150]
    tables, nb = tables_for(lens, 16, gen)
    pool = make_pool(nb, 16, 1, 64, gen, scales=(-8, -7))
    ref = RefPool(pool.storage, pool.scales)
    q = torch.randn((2, 4, 64), generator=gen) * 2.0 ** power
    s = 0.125 * 2.0 ** -power
    want, bound = ref.decode(q, tables, lens, s)
    out = pool.decode(q.to(DEV), tables, i32(lens), scale=s, max_ctx=150)
    assert ((out.cpu().double() - want).abs() <= bound).all()


def test_decode_large_scores():
    # one token outweighs the rest by hundreds of nats
    run_decode([100, 900], 16, 2, 4, 64, torch.float32, seed=23, scale=3.0)


def test_decode_many_light_tokens():
    # 20000 tokens 15 to 20 nats below one heavy token still add what they should
    gen = torch.Generator().manual_seed(41)
    n, bs, D = 20001, 32, 64
    tables, nb = tables_for([n], bs, gen)
    pool = make_pool(nb, bs, 1, D, gen, mass=True, scales=(-8, -7))
    raw = pool.storage.view(torch.uint8)
    raw[0] &= 0x9F  # small keys
    pos = 7777
    raw[0, int(tables[0, pos // bs]), 0, pos % bs] = 0x70  # 128 in every dim
    q = torch.full((1, 2, D), 0.25)
    ref = RefPool(pool.storage, pool.scales, pool.mass)
    want, bound = ref.decode(q, tables, [n], 2.2, accumulate=True)
    out = pool.decode(q.to(DEV), tables, i32([n]), scale=2.2, max_ctx=n, accumulate=True)
    assert ((out.cpu().double() - want).abs() <= bound).all()
    assert ((pool.mass.cpu().double() - ref.mass).abs() <= ref.mass_bound).all()


def test_decode_nan_in_a_key_is_that_sequences_own():
    gen = torch.Generator().manual_seed(51)
    lens = [50, 50]
    tables, nb = tables_for(lens, 16, gen)
    pool = make_pool(nb, 16, 1, 64, gen)
    pool.storage.view(torch.uint8)[0, int(tables[0, 1]), 0, 3, 5] = NAN_CODE
    out = pool.decode(torch.ones((2, 4, 64), device=DEV), tables, i32(lens), max_ctx=50)
    assert out[0].isnan().all() and out[1].isfinite().all()


def test_decode_any_positive_scales():
    # a loaded cache's scales need not be powers of two
    gen = torch.Generator().manual_seed(52)
    lens = [77, 130]
    tables, nb = tables_for(lens, 16, gen)
    pool = make_pool(nb, 16, 2, 128, gen)
    pool.scales.copy_(torch.rand(pool.scales.shape, generator=gen) * 0.02 + 1e-4)
    ref = RefPool(pool.storage, pool.scales)
    q = torch.randn((2, 8, 128), generator=gen)
    want, bound = ref.decode(q, tables, lens, 0.05)
    out = pool.decode(q.to(DEV), tables, i32(lens), scale=0.05, max_ctx=130)
    assert ((out.cpu().double() - want).abs() <= bound).all()


def test_decode_bad_tables_and_lengths_are_flagged():
    gen = torch.Generator().manual_seed(53)
    lens = [20, 40]
    tables, nb = tables_for(lens, 16, gen, width=4)
    pool = make_pool(nb, 16, 2, 64, gen, mass=True)
    q = torch.randn((2, 4, 64), generator=gen).to(DEV)
    bad = tables.clone()
    for v in (nb, 10 ** 6, -3):
        bad[1, 1] = v
        out = pool.decode(q, bad, i32(lens), max_ctx=40, accumulate=True)
        assert pool.pool_status() & _lib.FLAG_BLOCK_OOB
        kv = torch.randn((2, 2, 2, 64), generator=gen).to(DEV)
        pool.decode(q, bad, i32([20, 24]), max_ctx=40, k_new=kv[0], v_new=kv[1], accumulate=True)
        assert pool.pool_status() & _lib.FLAG_BLOCK_OOB
    out = pool.decode(q, tables, i32([20, 41]), max_ctx=40)
    assert pool.pool_status() == _lib.FLAG_CTX_RANGE and out.isfinite().all()
    out = pool.decode(q, tables, i32([-5, 40]), max_ctx=40)
    assert pool.pool_status() == _lib.FLAG_CTX_RANGE and (out[0] == 0).all()
    pool.decode(q, tables, i32(lens), max_ctx=40)
    assert pool.pool_status() == 0


def test_created_pool_is_clear_before_its_first_call():
    """The codes' and the index's zeros are written before create returns, not
    behind a call on a stream that does not wait for the creating one."""
    lib, h = _lib.lib(), C.c_void_p()
    nb, bs, H, D, n = 1 << 18, 16, 8, 64, 400
    gen = torch.Generator().manual_seed(55)
    kv = torch.randn((2, n, H, D), generator=gen).to(DEV)
    slots = torch.arange(n, dtype=torch.int32, device=DEV)
    table = torch.arange(n // bs, dtype=torch.int32, device=DEV)[None]
    out = torch.empty((2, n, H, D), device=DEV)
    ws = torch.empty(4 * n, dtype=torch.uint8, device=DEV)
    lens, s = i32([n]), torch.cuda.Stream()
    torch.cuda.synchronize()
    _lib.check(lib.clove_fp8_pool_create(0, nb, bs, H, D, 1, C.byref(h)))
    try:
        _lib.check(lib.clove_fp8_append(h, _lib.DTYPE_F32, kv[0].data_ptr(), kv[1].data_ptr(), slots.data_ptr(), n,
                                        ws.data_ptr(), 4 * n, s.cuda_stream))
        _lib.check(lib.clove_fp8_gather(h, table.data_ptr(), n // bs, lens.data_ptr(), 1, n, out[0].data_ptr(),
                                        out[1].data_ptr(), s.cuda_stream))
        s.synchronize()
        # half a step of e4m3 (2^-4), or of its subnormals: 2^-10 of a scale <= 2 max / 448
        assert ((out - kv).abs() <= kv.abs() * 2.0 ** -4 + kv.abs().max() * 2.0 ** -9 / 448).all()
    finally:
        lib.clove_fp8_pool_destroy(h)


@pytest.mark.parametrize("append", [False, True])
def test_decode_bad_tables_leave_other_weights_alone(append):
    gen = torch.Generator().manual_seed(54)
    pool = make_pool(8, 16, 2, 64, gen, mass=True)
    pool.mass.zero_()
    tables = torch.tensor([[3, 4, 5], [6, 99, -1]], dtype=torch.int32, device=DEV)
    q = torch.randn((2, 4, 64), generator=gen).to(DEV)
    kv = torch.randn((2, 2, 2, 64), generator=gen).to(DEV)
    new = dict(k_new=kv[0], v_new=kv[1]) if append else {}
    pool.decode(q, tables, i32([20, 40 - append]), max_ctx=40, accumulate=True, **new)
    assert pool.pool_status() == _lib.FLAG_BLOCK_OOB
    assert (pool.mass[[0, 1, 2, 7]] == 0).all() and (pool.mass[[3, 6]] > 0).all()


@pytest.mark.parametrize("shared", [3, 80])
def test_decode_forked_sequences_add_up_their_weights(shared):
    # forks read the same blocks in one call; each appends to a block of its own
    gen = torch.Generator().manual_seed(57)
    bs, H, D, B = 16, 2, 64, 6
    lens = [shared * bs + 5] * B
    tables = torch.zeros((B, shared + 1), dtype=torch.int32)
    tables[:, :shared] = torch.randperm(shared, generator=gen)
    tables[:, shared] = shared + torch.arange(B)
    tables = tables.to(DEV)
    pool = make_pool(shared + B, bs, H, D, gen, mass=True, scales=(-10, -6))
    ref = RefPool(pool.storage, pool.scales, pool.mass)
    q = torch.randn((B, 8, D), generator=gen)
    kv = torch.randn((2, B, H, D), generator=gen)
    ref.append(kv[0], kv[1], (shared + torch.arange(B)) * bs + 5)
    want, bound = ref.decode(q, tables, [n + 1 for n in lens], 0.125, accumulate=True)
    out = pool.decode(q.to(DEV), tables, i32(lens), scale=0.125, max_ctx=lens[0] + 1, k_new=kv[0].to(DEV),
                      v_new=kv[1].to(DEV), accumulate=True)
    assert ((out.cpu().double() - want).abs() <= bound).all()
    # B additions to one float32
    assert ((pool.mass.cpu().double() - ref.mass).abs() <= ref.mass_bound + B * 2.0 ** -23 * ref.mass).all()
    check_state(pool, ref)


def test_decode_empty_batch_and_no_tokens():
    pool = make_pool(4, 16, 2, 64, torch.Generator().manual_seed(54))
    out = torch.full((2, 4, 64), 7.0, device=DEV)
    pool.decode(torch.ones((2, 4, 64), device=DEV), i32([[0], [1]]), i32([0, 0]), max_ctx=0, out=out)
    assert (out == 0).all()
    pool.decode(torch.ones((0, 4, 64), device=DEV), i32([[0]])[:0], i32([]), max_ctx=4)


def test_decode_is_reproducible():
    gen = torch.Generator().manual_seed(55)
    lens = torch.randint(1, 3000, (40,), generator=gen).tolist()
    tables, nb = tables_for(lens, 16, gen)
    pool = make_pool(nb, 16, 4, 128, gen, mass=True)
    q = torch.randn((40, 16, 128), generator=gen).to(DEV)
    runs = []
    for _ in range(3):
        pool.mass.zero_()
        out = pool.decode(q, tables, i32(lens), max_ctx=max(lens), accumulate=True)
        runs.append((out.clone(), pool.mass.clone()))
    assert all(torch.equal(r[0], runs[0][0]) and torch.equal(r[1], runs[0][1]) for r in runs)


@pytest.mark.parametrize("lens", [[600, 40], [5000, 900]], ids=["whole", "split"])
def test_decode_stuck_wait_times_out_and_the_next_call_is_right(lens):
    # the test hook leaves one stage unfilled: its reader's bounded wait runs
    # out, the call ends and says so
    gen = torch.Generator().manual_seed(56)
    tables, nb = tables_for(lens, 16, gen)
    pool = make_pool(nb, 16, 2, 128, gen)
    ref = RefPool(pool.storage, pool.scales)
    q = torch.randn((2, 8, 128), generator=gen)
    L = _lib.lib()
    try:
        _lib.check(L.clove_cuda_debug_set(2000, 1))
        pool.decode(q.to(DEV), tables, i32(lens), max_ctx=max(lens))
        assert pool.pool_status() & _lib.FLAG_TIMEOUT
    finally:
        L.clove_cuda_debug_set(0, 0)
    want, bound = ref.decode(q, tables, lens, 128 ** -0.5)
    out = pool.decode(q.to(DEV), tables, i32(lens), max_ctx=max(lens))
    assert pool.pool_status() == 0
    assert ((out.cpu().double() - want).abs() <= bound).all()


# ---------------------------------------------------------------------------
# gather, copy
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("bs,H,D", [(8, 3, 64), (16, 2, 128), (128, 1, 256)])
def test_gather(bs, H, D):
    gen = torch.Generator().manual_seed(61)
    lens = [0, 1, bs, 3 * bs + 5]
    tables, nb = tables_for(lens, bs, gen)
    pool = make_pool(nb, bs, H, D, gen)
    poison(pool, tables, lens)
    ref = RefPool(pool.storage, pool.scales)
    got = pool.gather_kv(tables, i32(lens), max(lens))
    for p in range(2):
        for b, n in enumerate(lens):
            assert same(got[p][b, :n], ref.rows(p, tables[b].cpu(), torch.arange(n)))
            assert (got[p][b, n:] == 0).all()
    assert pool.pool_status() == 0


def test_copy_blocks():
    gen = torch.Generator().manual_seed(62)
    pool = make_pool(6, 16, 3, 64, gen, mass=True)
    before = (pool.storage.view(torch.uint8).clone(), pool.scales.clone(), pool.mass.clone())
    pool.copy_blocks(i32([0, 3, 5]), i32([1, 4, 5]))
    want = [0, 0, 2, 3, 3, 5]
    assert torch.equal(pool.storage.view(torch.uint8), before[0][:, want])
    assert torch.equal(pool.scales, before[1][:, want]) and torch.equal(pool.mass, before[2][want])
    pool.copy_blocks(i32([6, 0]), i32([2, -1]))
    assert pool.pool_status() == _lib.FLAG_BLOCK_OOB
    assert torch.equal(pool.mass, before[2][want])


# ---------------------------------------------------------------------------
# eviction
# ---------------------------------------------------------------------------
def run_evict(lens, bs, H, D, budget, recent, seed, values="random", scales=(-14, 1)):
    gen = torch.Generator().manual_seed(seed)
    tables, nb = tables_for([n for n in lens] + [min(n, budget) for n in lens], bs, gen,
                            width=max(1, (max(max(lens), 1) + bs - 1) // bs))
    old, new = tables[: len(lens)].contiguous(), tables[len(lens):].contiguous()
    pool = make_pool(nb, bs, H, D, gen, mass=True, scales=scales)
    if values == "ties":
        pool.mass.copy_(torch.randint(0, 3, pool.mass.shape, generator=gen).float())
    elif values == "equal":
        pool.mass.fill_(0.5)
    elif values == "wild":
        pool.mass.copy_(torch.exp(20 * torch.randn(pool.mass.shape, generator=gen)))
        flat = pool.mass.view(-1)
        flat[::7], flat[1::11], flat[2::13], flat[3::17] = 0.0, -0.0, float("inf"), float("nan")
        flat[5::19] = -1.0
        flat[6::23] = -float("nan")
    ref = RefPool(pool.storage, pool.scales, pool.mass)
    want = ref.evict(old, lens, new, budget, recent)
    kept, new_lens = pool.evict(old, i32(lens), new, budget, recent, max_ctx=max(lens))
    assert pool.pool_status() == 0
    assert torch.equal(new_lens.cpu(), want[1])
    assert torch.equal(kept.cpu(), want[0])
    check_state(pool, ref)
    assert same(pool.mass, ref.mass)


@pytest.mark.parametrize("bs,H,D", [(8, 2, 64), (16, 3, 128), (32, 1, 256), (256, 2, 64)])
@pytest.mark.parametrize("budget,recent", [(1, 0), (1, 1), (17, 0), (40, 40), (64, 10), (500, 100), (2000, 3)])
def test_evict(bs, H, D, budget, recent):
    run_evict([0, 1, 16, 41, 300, 1100], bs, H, D, budget, recent, seed=budget + recent + bs)


@pytest.mark.parametrize("values", ["ties", "equal", "wild"])
@pytest.mark.parametrize("budget,recent", [(100, 0), (700, 33)])
def test_evict_ties_and_odd_weights(values, budget, recent):
    run_evict([5, 1000, 2500, 1024], 16, 2, 64, budget, recent, seed=71, values=values)


def test_evict_long():
    run_evict([20000, 9000], 32, 1, 64, 3500, 100, seed=72)


def test_evict_scales_far_apart():
    run_evict([200, 77], 16, 2, 64, 50, 5, seed=73, scales=(-120, 100))


def test_evict_bad_tables_are_flagged():
    gen = torch.Generator().manual_seed(74)
    pool = make_pool(12, 16, 1, 64, gen, mass=True)
    old, new = i32([[0, 1, 2, 3]]), i32([[8, 9]])
    raw = pool.storage.view(torch.uint8).clone()
    pool.evict(i32([[0, 99, 2, -1]]), i32([64]), new, 32, 8, max_ctx=64)
    assert pool.pool_status() == _lib.FLAG_BLOCK_OOB
    pool.evict(old, i32([64]), i32([[12, -1]]), 32, 8, max_ctx=64)
    assert pool.pool_status() == _lib.FLAG_BLOCK_OOB
    keep = [i for i in range(12) if i not in (8, 9)]
    assert torch.equal(pool.storage.view(torch.uint8)[:, keep], raw[:, keep])
    _, lens = pool.evict(old, i32([70]), new, 32, 8, max_ctx=64)
    assert pool.pool_status() == _lib.FLAG_CTX_RANGE and lens.tolist() == [32]


# ---------------------------------------------------------------------------
# refusals
# ---------------------------------------------------------------------------
def test_refusals():
    from clove_b200 import Fp8KVPool
    pool = make_pool(8, 16, 2, 64, torch.Generator().manual_seed(81), mass=True)
    plain = Fp8KVPool(8, 16, 2, 64)
    assert plain.mass is None and (plain.scales == 0).all()
    bt, cl = i32([[0, 1], [2, 3]]), i32([20, 30])
    q = torch.randn((2, 4, 64), device=DEV)
    kv = torch.randn((2, 2, 64), device=DEV)
    ok = dict(max_ctx=32)
    for bad in (lambda: pool.decode(q.double(), bt, cl, **ok), lambda: pool.decode(q.cpu(), bt, cl, **ok),
                lambda: pool.decode(q, bt.long(), cl, **ok), lambda: pool.decode(q, bt, cl.cpu(), **ok),
                lambda: pool.decode(q, bt[:1], cl, **ok), lambda: pool.decode(q[:1], bt, cl, **ok),
                lambda: pool.decode(q, bt, cl, k_new=kv, **ok),
                lambda: pool.decode(q, bt, cl, k_new=kv, v_new=kv.half(), **ok),
                lambda: pool.decode(q, bt, cl, k_new=kv.half(), v_new=kv.half(), **ok),
                lambda: pool.decode(q, bt, cl, alibi_slopes=torch.ones(3, device=DEV), **ok),
                lambda: pool.decode(q, bt, cl, alibi_slopes=torch.ones(4), **ok),
                lambda: pool.decode(q, bt, cl, out=torch.empty((2, 4, 64), device=DEV).half(), **ok),
                lambda: plain.decode(q, bt, cl, accumulate=True, **ok),
                lambda: plain.evict(bt, cl, i32([[4], [5]]), 16),
                lambda: pool.evict(bt, cl, i32([[4], [5]]), 0), lambda: pool.evict(bt, cl, i32([[4], [5]]), 16, 17),
                lambda: pool.evict(bt, cl, i32([[4], [5]]), 16, -1), lambda: pool.evict(bt, cl, i32([[4]]), 16),
                lambda: pool.reshape_and_cache(kv, kv[:1], i32([0, 1])),
                lambda: pool.reshape_and_cache(kv, kv.half(), i32([0, 1])),
                lambda: pool.reshape_and_cache(kv, kv, torch.tensor([0, 1], device=DEV)),
                lambda: pool.gather_kv(bt, cl[:1], 32), lambda: pool.copy_blocks(i32([1, 2]), i32([3])),
                lambda: Fp8KVPool(8, 16, 2, 64, storage=pool.storage),
                lambda: Fp8KVPool(7, 16, 2, 64, storage=pool.storage, scales=pool.scales),
                lambda: Fp8KVPool(8, 16, 2, 64, mass=torch.zeros((8, 2, 8), device=DEV))):
        with pytest.raises(ValueError):
            bad()
    for code, bad in ((_lib.ERR_INVALID_ARG, lambda: pool.decode(q, bt, cl, max_ctx=33)),
                      (_lib.ERR_INVALID_ARG, lambda: pool.decode(q, bt, cl, max_ctx=-1)),
                      (_lib.ERR_INVALID_ARG, lambda: pool.decode(q[:, :3], bt, cl, **ok)),
                      (_lib.ERR_INVALID_ARG, lambda: pool.decode(q, bt, cl, softcap=-1.0, **ok)),
                      (_lib.ERR_INVALID_ARG, lambda: pool.decode(q, bt, cl, softcap=float("nan"), **ok)),
                      (_lib.ERR_INVALID_ARG, lambda: pool.decode(q, bt, cl, softcap=float("inf"), **ok)),
                      (_lib.ERR_INVALID_ARG, lambda: pool.decode(q, bt, cl, window=-1, **ok)),
                      (_lib.ERR_INVALID_ARG, lambda: pool.decode(q, bt, cl, k_new=kv, v_new=kv, max_ctx=0)),
                      (_lib.ERR_UNSUPPORTED, lambda: pool.decode(torch.ones((2, 18, 64), device=DEV), bt, cl, **ok)),
                      (_lib.ERR_INVALID_ARG, lambda: pool.evict(bt, cl, i32([[4], [5]]), 17, max_ctx=32)),
                      (_lib.ERR_UNSUPPORTED, lambda: Fp8KVPool(8, 4, 2, 64)),
                      (_lib.ERR_UNSUPPORTED, lambda: Fp8KVPool(8, 16, 2, 80))):
        with pytest.raises(_lib.CloveError) as e:
            bad()
        assert e.value.code == code
    assert pool.pool_status() == 0


def test_c_refusals_and_created_pool():
    L = _lib.lib()
    h = C.c_void_p()
    _lib.check(L.clove_fp8_pool_create(0, 16, 16, 2, 64, 1, C.byref(h)))
    info = _lib.Fp8PoolInfo()
    _lib.check(L.clove_fp8_pool_info(h, C.byref(info)))
    assert info.owns_memory == 1 and info.codes_bytes == 2 * 16 * 2 * 16 * 64 and info.mass and info.scales
    q = torch.ones((1, 4, 64), device=DEV)
    # a table wide enough for a call that needs scratch (a short one may not)
    bt, cl = i32([[0, 1] + [0] * 126]), i32([20])
    out = torch.empty((1, 4, 64), device=DEV)
    need = L.clove_fp8_decode_workspace_size(h, 1, 4, 2048, 0)
    assert need > 0
    ws = torch.empty(need + 256, dtype=torch.uint8, device=DEV)

    def decode(dtype=0, q=q.data_ptr(), k=None, v=None, out=out.data_ptr(), ws=ws.data_ptr(), n=need):
        return L.clove_fp8_decode(h, dtype, q, k, v, 4, bt.data_ptr(), 128, cl.data_ptr(), 1, 0.1, 2048, None, out, ws, n, None)

    assert decode() == 0
    torch.cuda.synchronize()
    assert (out == 0).all()  # a cache of zeros
    assert decode(dtype=32) == _lib.ERR_UNSUPPORTED
    assert decode(n=need - 1) == _lib.ERR_WORKSPACE and decode(ws=None) == _lib.ERR_WORKSPACE
    assert decode(ws=ws.data_ptr() + 16) == _lib.ERR_WORKSPACE
    assert decode(q=q.data_ptr() + 4) == -1 and decode(out=None) == -1 and decode(k=q.data_ptr()) == -1
    assert L.clove_fp8_append(h, 0, q.data_ptr() + 8, q.data_ptr(), cl.data_ptr(), 1, None, 0, None) == -1
    assert L.clove_fp8_evict(h, bt.data_ptr(), 2, cl.data_ptr(), 1, 33, bt.data_ptr(), 2, 16, 0, bt.data_ptr(),
                             cl.data_ptr(), None, 0, None) == -1
    _lib.check(L.clove_fp8_pool_destroy(h))


# ---------------------------------------------------------------------------
# streams, graphs, and the operators together
# ---------------------------------------------------------------------------
def test_decode_on_another_stream():
    gen = torch.Generator().manual_seed(91)
    lens = [900, 40]
    tables, nb = tables_for(lens, 16, gen)
    pool = make_pool(nb, 16, 2, 128, gen)
    q = torch.randn((2, 8, 128), generator=gen).to(DEV)
    cl = i32(lens)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    a = pool.decode(q, tables, cl, max_ctx=900, stream=side)
    with torch.cuda.stream(side):
        b = pool.decode(q, tables, cl, max_ctx=900)
    torch.cuda.synchronize()
    c = pool.decode(q, tables, cl, max_ctx=900)
    assert torch.equal(a, b) and torch.equal(a, c)


def test_two_captured_graphs_at_once():
    # two steps over different sequences of one pool, captured apart and
    # replayed at the same time on two streams
    gen = torch.Generator().manual_seed(92)
    bs, H, D, B = 16, 2, 128, 6
    lens = [[700, 33, 16, 5, 250, 90], [64, 900, 1, 31, 400, 77]]
    tables, nb = tables_for([n + 8 for n in lens[0] + lens[1]], bs, gen)
    pool = make_pool(nb, bs, H, D, gen, mass=True)
    ref = RefPool(pool.storage, pool.scales, pool.mass)
    q = torch.randn((2, B, 8, D), generator=gen)
    kv = torch.randn((2, 2, B, H, D), generator=gen)
    graphs, outs, held = [], [], []
    for i in range(2):
        t, cl = tables[i * B:(i + 1) * B].contiguous(), i32(lens[i])
        args = (q[i].to(DEV), t, cl)
        kw = dict(max_ctx=max(lens[i]) + 8, k_new=kv[i, 0].to(DEV), v_new=kv[i, 1].to(DEV), accumulate=True)
        g = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g):
            outs.append(pool.decode(*args, **kw))
            cl += 1
        graphs.append(g)
        held.append((args, kw))
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(4):
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for step in range(4):
        for i in range(2):
            t = tables[i * B:(i + 1) * B]
            now = [n + step for n in lens[i]]
            slots = torch.tensor([int(t[b, n // bs]) * bs + n % bs for b, n in enumerate(now)])
            ref.append(kv[i, 0], kv[i, 1], slots)
            want, bound = ref.decode(q[i], t, [n + 1 for n in now], D ** -0.5, accumulate=True)
            if step == 3:
                assert ((outs[i].cpu().double() - want).abs() <= bound).all()
    check_state(pool, ref)
    assert pool.pool_status() == 0


def test_captured_append_and_evict():
    gen = torch.Generator().manual_seed(93)
    pool = make_pool(120, 16, 2, 64, gen, mass=True)
    slots = i32(torch.randperm(100 * 16, generator=gen)[:1500])
    kv = torch.randn((2, 1500, 2, 64), generator=gen).to(DEV)
    old, new, lens = i32(torch.arange(100).reshape(2, 50)), i32([[100, 101, 102], [103, 104, 105]]), i32([800, 600])
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        pool.reshape_and_cache(kv[0], kv[1], slots)
        kept, new_lens = pool.evict(old, lens, new, 40, 8, max_ctx=800)
    for _ in range(2):  # the second replay starts from what the first left
        before = RefPool(pool.storage, pool.scales, pool.mass)
        pool.mass.copy_(torch.rand(pool.mass.shape, generator=gen))
        before.mass = pool.mass.cpu().double()
        g.replay()
        torch.cuda.synchronize()
        before.append(kv[0], kv[1], slots)
        want = before.evict(old, [800, 600], new, 40, 8)
        assert torch.equal(kept.cpu(), want[0]) and new_lens.tolist() == [40, 40]
        check_state(pool, before)


def test_serving_run():
    # prompts, decode steps that add up weights, an eviction into new blocks
    # of the block manager, and further steps over the smaller cache
    from clove_b200 import Fp8KVPool
    from clove_b200.blocks import BlockManager
    gen = torch.Generator().manual_seed(94)
    B, H, G, D, bs, nb, stride = 3, 2, 4, 128, 16, 64, 16
    mgr, pool = BlockManager(nb, bs, 8), Fp8KVPool(nb, bs, H, D, track_mass=True)
    ref = RefPool(pool.storage, pool.scales, pool.mass)
    prompt = [37, 120, 5]

    def rand(*shape):
        return torch.randn(shape, generator=gen).bfloat16()

    def step(seqs, softcap):
        for s in seqs:
            assert mgr.reserve(s, mgr.seq_len(s) + 1) == []
        t, n = mgr.export(seqs, stride)
        lens = torch.from_numpy(n) - 1
        q, k, v = rand(B, H * G, D), rand(B, H, D), rand(B, H, D)
        tables = torch.from_numpy(t)
        out = pool.append_decode(q.to(DEV), k.to(DEV), v.to(DEV), tables.to(DEV), i32(lens), max_ctx=int(n.max()),
                                 softcap=softcap, accumulate=True)
        ref.append(k, v, torch.tensor([int(tables[b, x // bs]) * bs + x % bs for b, x in enumerate(lens.tolist())]))
        want, bound = ref.decode(q, tables, n.tolist(), D ** -0.5, softcap, accumulate=True)
        assert ((out.cpu().double() - want).abs() <= bound).all()

    for s, n in enumerate(prompt):
        mgr.add(s, n)
    t, _ = mgr.export(range(B), stride)
    slots = torch.cat([torch.from_numpy(t[b]).long()[torch.arange(n) // bs] * bs + torch.arange(n) % bs
                       for b, n in enumerate(prompt)])
    k, v = rand(sum(prompt), H, D), rand(sum(prompt), H, D)
    pool.reshape_and_cache(k.to(DEV), v.to(DEV), i32(slots))
    ref.append(k, v, slots)
    for _ in range(6):
        step([0, 1, 2], 30.0)
    check_state(pool, ref)
    budget = 24
    t, n = mgr.export([0, 1, 2], stride)
    for s, x in enumerate(n.tolist()):
        mgr.add(4 + s, min(x, budget))
    new, _ = mgr.export([4, 5, 6], stride)
    ref.mass = pool.mass.cpu().double()  # the choice goes by the weights as the pool holds them
    want = ref.evict(torch.from_numpy(t), n.tolist(), torch.from_numpy(new), budget, 8)
    kept, lens = pool.evict(i32(t), i32(n), i32(new), budget, 8, max_ctx=int(n.max()))
    assert torch.equal(kept.cpu(), want[0]) and torch.equal(lens.cpu(), want[1])
    for s in range(3):
        mgr.free(s)
    for _ in range(10):
        step([4, 5, 6], 30.0)
    check_state(pool, ref)
    assert pool.pool_status() == 0


def test_prefilled_16_bit_blocks_move_over():
    # a prompt prefilled in a 16-bit pool, gathered and quantised
    from clove_b200 import Fp8KVPool, KVPool
    gen = torch.Generator().manual_seed(95)
    n, bs, H, D = 70, 16, 2, 128
    src = KVPool(8, bs, H, D, torch.bfloat16, 0)
    q, k, v = (torch.randn((n, h, D), generator=gen).bfloat16().to(DEV) for h in (4, H, H))
    bt, zero = i32([[3, 1, 6, 0, 5]]), i32([0])
    src.prefill(q, k, v, i32([0, n]), bt, zero, max_ctx=n, rope_theta=10000.0)
    kg, vg = src.gather_kv(bt, i32([n]), n)
    pool = Fp8KVPool(8, bs, H, D)
    ref = RefPool(pool.storage, pool.scales)
    slots = torch.arange(n) + 16
    pool.reshape_and_cache(kg[0], vg[0], i32(slots))
    ref.append(kg[0], vg[0], slots)
    check_state(pool, ref)


def test_module_step_over_the_8_bit_cache():
    from clove_b200 import Fp8KVPool
    from clove_b200.backend import PagedAttention
    B, dim, heads, kvh, bs = 3, 256, 4, 2, 16
    att = PagedAttention(dim, heads, kvh, device=DEV, seed=3)
    pool = Fp8KVPool(12, bs, kvh, dim // heads)
    gen = torch.Generator().manual_seed(96)
    x = torch.randn((B, dim), generator=gen).to(DEV)
    bt, cl = i32([[0, 1], [2, 3], [4, 5]]), i32([0, 16, 20])
    k0 = torch.randn((36, kvh, dim // heads), generator=gen).to(DEV)
    pool.reshape_and_cache(k0, k0, i32(list(range(32, 48)) + list(range(64, 84))))
    ref = RefPool(pool.storage, pool.scales)
    y = att.forward(x, pool, bt, cl, max_ctx=21)
    q, k, v = att.w_q.forward(x), att.w_k.forward(x), att.w_v.forward(x)
    ref.append(k.reshape(B, kvh, -1), v.reshape(B, kvh, -1), torch.tensor([0, 48, 84]))
    want, bound = ref.decode(q.reshape(B, heads, -1), bt, [1, 17, 21], (dim // heads) ** -0.5)
    check_state(pool, ref)
    w = att.w_o.weight.cpu().double()
    off = (y.cpu().double() - want.reshape(B, -1) @ w).abs()
    # the projection adds dim products in float32
    assert (off <= bound.reshape(B, -1) @ w.abs() + dim * 2.0 ** -24 * (want.reshape(B, -1).abs() @ w.abs())).all()
    with pytest.raises(TypeError):
        att.forward_fused(x, pool, bt, cl, max_ctx=21)
