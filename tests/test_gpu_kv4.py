"""The 4-bit KV cache's kernels against the float64 checker (needs an MI355X).

Bounds, derived from how the kernels compute (u = 2^-24; a rounding to t is off by at most
finfo(t).eps / 2 relative):
  cached codes and scales   equal: keys are rotated in double and rounded once
  rotated queries           two products and a sum: 2 u (|x cos| + |y sin|), and the rounding to the dtype
  angles                    the float's rounding, and 2^-52 |angle| for the double product
  attention                 scores: a dot product of D exact products in up to three pieces, accumulated in
                            float: (3 D + 8) u S with S the largest sum |q| |k| |scale|; a score error d moves
                            a softmax weight by 2 d; the weights enter the second product with 2^-8 (bf16),
                            2^-16 (fp16) or 2^-24 (fp32); exp2 and the n-term sums add 2^-22 + 2 (n + 8) u.
                            All of that times the weighted mean of |v|, plus the rounding of the result.
"""
import math

import numpy as np
import pytest
import torch

from oracle import kv4_oracle as orc

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
WEIGHT = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -16, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}      # half a subnormal step
ALL = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(scope='module')
def ops(device):
    from mi355_paged import ops
    return ops


def _cast(x, dtype):
    """float64 numpy -> (device tensor of dtype, its values in float64)."""
    t = torch.from_numpy(np.asarray(x)).to(dtype)
    return t.cuda(), t.double().numpy()


def _near(got, want, bound):
    got = got.double().cpu().numpy()
    bad = ~(np.abs(got - want) <= bound)
    assert not bad.any(), (f"{bad.sum()} of {bad.size} off, first at {np.argwhere(bad)[0]}: {got[bad][:4]} for {want[bad][:4]}, "
                           f"allowed {np.broadcast_to(bound, want.shape)[bad][:4]}")


# ------------------------------------------------------------------ angles
@pytest.mark.parametrize('T,half', [(1, 8), (3, 1), (77, 24), (1025, 64)])
def test_angles(ops, device, T, half):
    rng = np.random.default_rng(T + half)
    pos = rng.integers(0, 1 << 22, T)
    pos[0] = 0
    if T > 5:
        pos[1:6] = [1, 8191, (1 << 31) + 5, (1 << 40) + 1, -7]
    freq, factor = ops.rope_frequencies(2 * half, scaling={'kind': 'yarn', 'factor': 8, 'original': 4096})
    cos, sin = ops.rope_angles(torch.from_numpy(pos).cuda(), freq.cuda(), factor)
    assert cos.dtype == sin.dtype == torch.float32 and cos.shape == sin.shape == (T, half)
    a = pos[:, None].astype(np.float64) * freq.numpy()
    for got, want in ((cos, np.cos(a) * factor), (sin, np.sin(a) * factor)):
        _near(got, want, U * np.abs(want) + factor * (2.0 ** -52 * np.abs(a) + 2e-11))


@pytest.mark.parametrize('kind', [None, 'yarn'])
def test_angles_of_far_positions(ops, device, kind):
    """cos and sin of the rounded product itself, up to the last position: the first Taylor term left out, (pi/4)^13 / 13! =
    7e-12, and the rounding to float."""
    rng = np.random.default_rng(5)
    pos = np.concatenate([rng.integers(1 << e, 1 << (e + 1), 40) for e in range(63)] + [np.array([0, (1 << 53) + 1, (1 << 63) - 1, -(1 << 63)])])
    pos[::7] *= -1
    freq, factor = ops.rope_frequencies(64, scaling=kind and {'kind': kind, 'factor': 8, 'original': 4096})
    cos, sin = ops.rope_angles(torch.from_numpy(pos).cuda(), freq.cuda(), factor)
    a = pos[:, None].astype(np.float64) * freq.numpy()
    for got, f in ((cos, math.cos), (sin, math.sin)):
        want = np.vectorize(f)(a) * factor
        _near(got, want, U * np.abs(want) + factor * 7.1e-12)
    cos, sin = ops.rope_angles(torch.tensor([1, (1 << 63) - 1], device=device), torch.tensor([1e300, 4.0, 1.0], dtype=torch.float64, device=device))
    assert torch.isnan(cos).tolist() == torch.isnan(sin).tolist() == [[True, False, False], [True, True, False]]


def test_angles_refusals(ops, device):
    pos, freq = torch.zeros(3, dtype=torch.int64, device=device), torch.ones(4, dtype=torch.float64, device=device)
    with pytest.raises(TypeError):
        ops.rope_angles(pos.int(), freq)
    with pytest.raises(TypeError):
        ops.rope_angles(pos, freq.float())
    cos, sin = ops.rope_angles(pos[:0], freq)
    assert cos.shape == (0, 4)


# ------------------------------------------------------------------ rotation and append
def _rows(rng, T, Hq, Hkv, D, dtype):
    """q, k, v as views of one projection output, and their values."""
    x = rng.standard_normal((T, (Hq + 2 * Hkv) * D)) * np.exp2(rng.integers(-3, 4, (Hq + 2 * Hkv) * D))
    t, val = _cast(x, dtype)
    cut = [Hq * D, Hkv * D, Hkv * D]
    views = [c.view(T, -1, D) for c in t.split(cut, -1)]
    vals = [c.reshape(T, -1, D) for c in np.split(val, np.cumsum(cut)[:-1], -1)]
    return views, vals


def _angle_rows(ops, rng, T, R):
    if R == 0:
        return None, None, np.zeros((T, 0)), np.zeros((T, 0))
    freq, _ = ops.rope_frequencies(R)
    cos, sin = ops.rope_angles(torch.from_numpy(rng.integers(0, 100000, T)).cuda(), freq.cuda())
    return cos, sin, cos.double().cpu().numpy(), sin.double().cpu().numpy()


def _rotation_bound(x, cos, sin, inter, dtype, want):
    size = orc.rotate(np.abs(x), np.abs(cos), -np.abs(sin), inter)      # |a c| + |b s| for the first of a pair
    other = orc.rotate(np.abs(x), np.abs(cos), np.abs(sin), inter)      # ... and for the second
    return 2 * U * np.maximum(np.abs(size), np.abs(other)) * (1 + HALF[dtype]) + HALF[dtype] * np.abs(want) + TINY[dtype]


@pytest.mark.parametrize('dtype', ALL)
@pytest.mark.parametrize('T,Hq,Hkv,D,BS,R,inter', [
    (1, 8, 8, 64, 16, 64, False), (37, 8, 2, 128, 16, 128, True), (50, 4, 4, 32, 32, 16, False), (19, 6, 3, 256, 48, 64, True),
    (64, 7, 1, 64, 64, 32, False), (300, 2, 2, 32, 16, 32, True), (33, 3, 3, 128, 16, 0, False)])
def test_append_rounds_rotates_and_scatters(ops, device, dtype, T, Hq, Hkv, D, BS, R, inter):
    rng = np.random.default_rng(T * 1000 + D + Hq)
    (q, k, v), (qv, kv, vv) = _rows(rng, T, Hq, Hkv, D, dtype)
    cos, sin, cv, sv = _angle_rows(ops, rng, T, R)
    NB = -(-T // BS) + 3
    slots = rng.permutation(NB * BS)[:T]
    if T > 4:
        slots[2], slots[4] = -1, NB * BS                       # skipped
    old = [rng.integers(0, 256, ops.kv4_cache_shape(NB, Hkv, BS, D)).astype(np.uint8) for _ in range(2)]
    kc, vc = (torch.from_numpy(o).cuda() for o in old)
    before = [t.clone() for t in (q, k, v)]
    out = ops.rope_kv4_write(q, k, v, cos, sin, torch.from_numpy(slots).cuda(), kc, vc, interleaved=inter)
    assert all(torch.equal(a, b) for a, b in zip(before, (q, k, v)))
    want = orc.rotate(qv, cv, sv, inter)
    _near(out, want, _rotation_bound(qv, cv, sv, inter, dtype, want))
    want = [old[0].copy(), old[1].copy()]
    for form, x in enumerate((orc.rotate(kv, cv, sv, inter), vv)):
        code, byte = orc.quantise(x)
        for t in range(T):
            if 0 <= slots[t] < NB * BS:
                blk, at = divmod(int(slots[t]), BS)
                for h in range(Hkv):
                    orc.write_row(want[form][blk, h, at // 16], at % 16, code[t, h], byte[t, h], bool(form))
    for got, w in ((kc, want[0]), (vc, want[1])):
        np.testing.assert_array_equal(got.cpu().numpy(), w)    # written rows and every byte beside them
    # the same rows read back, at an invalid slot zeros
    rk, rv = ops.kv4_read_slots(kc, vc, torch.from_numpy(slots).cuda(), torch.float32)
    for form, got in enumerate((rk, rv)):
        for t in range(T):
            if 0 <= slots[t] < NB * BS:
                blk, at = divmod(int(slots[t]), BS)
                values = orc.unpack(want[form][blk, :, at // 16], bool(form))[:, at % 16]
                np.testing.assert_array_equal(got[t].double().cpu().numpy(), values)
            else:
                assert not got[t].any()


@pytest.mark.parametrize('dtype', ALL)
@pytest.mark.parametrize('T,Hq,Hkv,D,BS,R,inter', [(12301, 4, 8, 64, 16, 64, False), (3075, 2, 8, 256, 48, 128, True),
                                                   (24601, 1, 8, 32, 32, 32, False), (6145, 3, 8, 128, 16, 0, False)])
def test_append_and_read_of_many_rows_equal_those_of_few(ops, device, dtype, T, Hq, Hkv, D, BS, R, inter):
    """A call long enough for two tokens per thread gives the bytes and values of short calls (which the test above
    holds against the oracle): slots in runs of either parity, scattered, backwards and outside the cache."""
    rng = np.random.default_rng(T)
    (q, k, v), _ = _rows(rng, T, Hq, Hkv, D, dtype)
    cos, sin, _, _ = _angle_rows(ops, rng, T, R)
    NB = -(-T // BS) + 9
    slots = np.arange(T) + 7
    slots[1000:1501] = slots[1000:1501][rng.permutation(501)]
    slots[1600:1701] = slots[1600:1701][::-1]
    slots[2001:3001] = np.roll(slots[2001:3001], 1)
    slots[[5, 900, 901, T - 1]] = [-1, NB * BS, NB * BS + 1, -2]
    slots = torch.from_numpy(slots).cuda()
    caches = [[torch.full(ops.kv4_cache_shape(NB, Hkv, BS, D), 90, dtype=torch.uint8, device=device) for _ in range(2)] for _ in range(2)]
    whole = ops.rope_kv4_write(q, k, v, cos, sin, slots, *caches[0], interleaved=inter)
    rk, rv = ops.kv4_read_slots(*caches[0], slots, dtype)
    for a in range(0, T, 500):
        b = min(a + 500, T)
        part = ops.rope_kv4_write(q[a:b], k[a:b], v[a:b], *((cos[a:b], sin[a:b]) if R else (None, None)), slots[a:b], *caches[1],
                                  interleaved=inter)
        assert torch.equal(whole[a:b], part)
    for a in range(0, T, 500):
        pk, pv = ops.kv4_read_slots(*caches[1], slots[a:a + 500], dtype)
        assert torch.equal(rk[a:a + 500], pk) and torch.equal(rv[a:a + 500], pv)
    assert torch.equal(caches[0][0], caches[1][0]) and torch.equal(caches[0][1], caches[1][1])


def test_append_values_at_borders_extremes_and_nan(ops, device):
    D, T = 64, 9
    x = np.zeros((T, 1, D))
    x[0, 0, :16] = [6, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, -0.25, -0.75, -5, 0.2500001, 0.7499999, 4.9999995, 5.0000005, -0.0]
    x[1, 0, :4] = [3.4e38, 1.0, -3.4e38, 1e30]                 # saturates at 6 * 2^125
    x[2, 0, :4] = [1e-38, 1e-40, -1e-36, 2e-36]                # below the smallest scale
    x[3, 0, 5] = np.nan
    x[4, 0, 40] = np.inf                                       # only its own block of 32 reads as NaN
    x[5, 0, :3] = [6.0000005, 1, 2]
    x[6] = 0.0
    x[7, 0, :32] = 2.0 ** -126
    x[8, 0, 33] = -np.inf
    t, val = _cast(x, torch.float32)
    kc, vc = (torch.zeros(ops.kv4_cache_shape(1, 1, 16, D), dtype=torch.uint8, device=device) for _ in range(2))
    out = ops.rope_kv4_write(t, t, t, None, None, torch.arange(T, device=device), kc, vc)
    assert torch.equal(out.view(torch.int32), t.view(torch.int32))
    code, byte = orc.quantise(val)
    want = orc.dequantise(code, byte)
    rk, rv = ops.kv4_read_slots(kc, vc, torch.arange(T, device=device), torch.float32)
    np.testing.assert_array_equal(rk.double().cpu().numpy(), want)
    np.testing.assert_array_equal(rv.double().cpu().numpy(), want)
    half, _ = ops.kv4_read_slots(kc, vc, torch.arange(1, device=device), torch.float16)
    np.testing.assert_array_equal(half.double().cpu().numpy(), want[:1])


@pytest.mark.parametrize('dtype', ALL)
@pytest.mark.parametrize('T,H,D,R,inter', [(1, 1, 32, 32, False), (41, 5, 64, 48, True), (7, 3, 256, 128, False), (9, 2, 128, 0, False)])
def test_rotate(ops, device, dtype, T, H, D, R, inter):
    rng = np.random.default_rng(T + R)
    wide, val = _cast(rng.standard_normal((T, (H + 1) * D)), dtype)
    x, xv = wide[:, D:].view(T, H, D), val[:, D:].reshape(T, H, D)
    cos, sin, cv, sv = _angle_rows(ops, rng, T, R)
    want = orc.rotate(xv, cv, sv, inter)
    out = torch.full((T, H, D), math.nan, dtype=dtype, device=device)
    assert ops.rope_rotate(x, cos, sin, inter, out=out) is out
    _near(out, want, _rotation_bound(xv, cv, sv, inter, dtype, want))
    assert torch.equal(out[..., R:], x[..., R:])


def test_append_refusals(ops, device):
    kc, vc = (torch.zeros(ops.kv4_cache_shape(4, 2, 16, 64), dtype=torch.uint8, device=device) for _ in range(2))
    x = torch.zeros(3, 2, 64, device=device, dtype=torch.bfloat16)
    cs = torch.zeros(3, 32, device=device)
    slots = torch.arange(3, device=device)
    for bad in (dict(k=x[:2]), dict(v=x[:, :1]), dict(k_cache=kc[:2]), dict(slots=slots[:2].int()), dict(slots=slots[:2]),
                dict(cos=None), dict(cos=cs[:2], sin=cs[:2]), dict(cos=cs.double(), sin=cs.double()), dict(q=x.float()),
                dict(q=torch.zeros(3, 2, 128, device=device, dtype=torch.bfloat16)), dict(k_cache=kc.int(), v_cache=vc.int()),
                dict(out=torch.empty(3, 2, 64, device=device)), dict(q=x.transpose(0, 1)),
                dict(k_cache=kc[..., :500], v_cache=vc[..., :500])):
        args = dict(q=x, k=x, v=x, cos=cs, sin=cs, slots=slots, k_cache=kc, v_cache=vc)
        with pytest.raises((TypeError, ValueError)):
            ops.rope_kv4_write(**dict(args, **bad))
    from mi355_paged._lib import Mi355Error
    odd = torch.zeros(3 * 128 + 1, device=device, dtype=torch.bfloat16)[1:].view(3, 2, 64)
    with pytest.raises(Mi355Error, match='aligned'):
        ops.rope_kv4_write(odd, x, x, cs, cs, slots, kc, vc)
    with pytest.raises(Mi355Error, match='rotary_dim'):
        ops.rope_rotate(x, cs[:, :12].contiguous(), cs[:, :12].contiguous())
    assert ops.rope_kv4_write(x[:0], x[:0], x[:0], cs[:0], cs[:0], slots[:0], kc, vc).shape == (0, 2, 64)


# ------------------------------------------------------------------ caches for the attention tests
def _cache(rng, lens, Hkv, D, BS, spare=2, fill=255):
    """(K records, V records, block tables) of sequences with `lens` cached tokens; rows nobody wrote hold `fill`."""
    need = [-(-n // BS) for n in lens]
    NB = sum(need) + spare
    order = rng.permutation(NB)
    width = max(max(need), 1)
    tables = np.full((len(lens), width), NB + 7, dtype=np.int32)     # entries nobody may follow
    caches = []
    at = 0
    for i, n in enumerate(need):
        tables[i, :n] = order[at:at + n]
        at += n
    for form in (False, True):
        x = rng.standard_normal((NB, Hkv, BS // 16, 16, D)) * np.exp2(0.5 * rng.standard_normal(D))
        rec = orc.pack(*orc.quantise(x), form)
        empty = np.full(orc.record_bytes(D), fill, dtype=np.uint8)
        used = np.zeros((NB, BS), dtype=bool)
        for i, n in enumerate(lens):
            for t in range(n):
                used[tables[i, t // BS], t % BS] = True
        for blk in range(NB):
            for t in range(BS):
                if not used[blk, t]:
                    for h in range(Hkv):
                        r = rec[blk, h, t // 16]
                        for d in range(D):
                            a, s = orc.code_place(D, t % 16, d, form)
                            r[a] = (int(r[a]) & (0xF0 >> s)) | (int(empty[a]) & (15 << s))
                        for b in range(D // 32):
                            r[orc.scale_place(D, t % 16, b, form)] = fill
        caches.append(rec)
    return caches[0], caches[1], tables


def _attend_all(q, kc, vc, tables, lens, scale, limits):
    """q [rows of one sequence each: list of [n, Hq, D]]; limits [list of [n]] -> out, size, big as lists."""
    res = []
    for i, (qi, lim) in enumerate(zip(q, limits)):
        Hkv, Hq = kc.shape[1], qi.shape[1]
        G = Hq // Hkv
        o, s, b = np.zeros(qi.shape), np.zeros(qi.shape), np.zeros(qi.shape[:2] + (1,))
        for h in range(Hkv):
            if lens[i] == 0:
                continue
            k, v = orc.gather(kc, tables[i], lens[i], h, False), orc.gather(vc, tables[i], lens[i], h, True)
            for g in range(G):
                o[:, h * G + g], s[:, h * G + g], b[:, h * G + g] = orc.attend(qi[:, h * G + g], k, v, scale, lim)
        res.append((o, s, b))
    return [np.concatenate([r[j] for r in res]) for j in range(3)]


def _attention_bound(size, big, want, D, n, dtype):
    return (2 * (3 * D + 8) * U * big + 2.0 ** -22 + 2 * (n + 8) * U + WEIGHT[dtype]) * size + \
        (HALF[dtype] + 2 * (n + 8) * U) * np.abs(want) + 1e-30


DECODE = [
    # Hq, Hkv, D, BS, context lengths
    (8, 8, 64, 16, [1, 2, 15, 16, 17, 0, 31, 32, 33, 37]),
    (8, 8, 32, 32, [127, 128, 129, 1, 0, 200]),
    (32, 8, 128, 16, [50, 257]),
    (14, 2, 64, 48, [300, 7, 48]),
    (6, 6, 256, 16, [65, 16]),
    (3, 3, 64, 16, [140]),
    (16, 1, 128, 64, [33, 500]),
    (20, 1, 64, 16, [70]),
    (40, 2, 32, 16, [90, 3]),
    (8, 4, 256, 16, [20]),
    (5, 5, 128, 16, [0, 0]),
    (8, 8, 64, 16, [1900, 40]),
]


@pytest.mark.parametrize('dtype', ALL)
@pytest.mark.parametrize('Hq,Hkv,D,BS,lens', DECODE, ids=lambda v: str(v))
def test_decode(ops, device, dtype, Hq, Hkv, D, BS, lens):
    rng = np.random.default_rng(Hq * 131 + D + sum(lens))
    kc, vc, tables = _cache(rng, lens, Hkv, D, BS)
    B = len(lens)
    wide, val = _cast(rng.standard_normal((B, (Hq + 1) * D)) * 1.5, dtype)
    q, qv = wide[:, D:].view(B, Hq, D), val[:, D:].reshape(B, Hq, D)
    scale = D ** -0.5
    want, size, big = _attend_all([qv[i:i + 1] for i in range(B)], kc, vc, tables, lens, scale, [[n - 1] for n in lens])
    out = ops.paged_decode_kv4(q, torch.from_numpy(kc).cuda(), torch.from_numpy(vc).cuda(), torch.from_numpy(tables).cuda(),
                               torch.tensor(lens, dtype=torch.int32, device=device), max(lens))
    _near(out, want, _attention_bound(size, big, want, D, max(lens), dtype))
    for i, n in enumerate(lens):
        if n == 0:
            assert not out[i].any()


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
def test_decode_long_context_split_and_bounds(ops, device, dtype):
    """Many splits (some of them empty), a max_context far above and one below the contexts."""
    rng = np.random.default_rng(3)
    lens, Hq, Hkv, D, BS = [9001, 130, 0, 4097], 4, 2, 64, 16
    kc, vc, tables = _cache(rng, lens, Hkv, D, BS)
    q, qv = _cast(rng.standard_normal((4, Hq, D)), dtype)
    args = [torch.from_numpy(a).cuda() for a in (kc, vc, tables)]
    ctx = torch.tensor(lens, dtype=torch.int32, device=device)
    for bound in (9001, 100000, 4100):
        seen = [min(n, bound) for n in lens]
        want, size, big = _attend_all([qv[i:i + 1] for i in range(4)], kc, vc, tables, seen, D ** -0.5, [[n - 1] for n in seen])
        out = ops.paged_decode_kv4(q, *args, ctx, bound)
        _near(out, want, _attention_bound(size, big, want, D, max(lens), dtype))
    again = ops.paged_decode_kv4(q, *args, ctx, 4100)
    assert torch.equal(again, out)


@pytest.mark.parametrize('dtype', ALL)
@pytest.mark.parametrize('B,Hq,Hkv,D,longest', [(256, 8, 8, 64, 520), (256, 32, 8, 64, 257), (128, 8, 8, 128, 530), (257, 8, 8, 32, 1030),
                                                (90, 16, 8, 32, 3000), (8, 8, 4, 128, 20000)])
def test_decode_of_many_sequences(ops, device, dtype, B, Hq, Hkv, D, longest):
    """Enough work for several kv heads per wave: six sequences against the oracle, a NaN block in one of them."""
    rng = np.random.default_rng(B + D)
    BS, G = 16, Hq // Hkv
    lens = rng.integers(1, longest + 1, B)
    lens[[0, B - 1]] = [longest, 1]
    need = -(-lens // BS)
    order = rng.permutation(int(need.sum()) + 3)
    tables = np.zeros((B, int(need.max())), dtype=np.int32)
    for i, at in enumerate(np.cumsum(need) - need):
        tables[i, :need[i]] = order[at:at + need[i]]
    shape = ops.kv4_cache_shape(len(order), Hkv, BS, D)
    kc, vc = (rng.integers(0, 256, shape, dtype=np.uint8) for _ in range(2))
    for c in (kc, vc):
        c[..., 8 * D:] = rng.integers(124, 128, shape[:-1] + (D // 2,), dtype=np.uint8)
    at = int(lens[0]) // 2
    vc[tables[0, at // BS], 1, 0, orc.scale_place(D, at % 16, 0, True)] = 255
    q, qv = _cast(rng.standard_normal((B, Hq, D)), dtype)
    out = ops.paged_decode_kv4(q, *(torch.from_numpy(a).cuda() for a in (kc, vc, tables)),
                               torch.tensor(lens, dtype=torch.int32, device=device), longest)
    nan = torch.isnan(out).cpu().numpy()
    assert nan[0, G:2 * G, :32].all() and nan.sum() == G * 32
    pick = [1, 2, B // 3, B // 2, B - 2, B - 1]
    want, size, big = _attend_all([qv[i:i + 1] for i in pick], kc, vc, tables[pick], [int(lens[i]) for i in pick], D ** -0.5,
                                  [[int(lens[i]) - 1] for i in pick])
    _near(out[pick], want, _attention_bound(size, big, want, D, longest, dtype))
    want, size, big = _attend_all([qv[:1, :G]], kc[:, :1], vc[:, :1], tables[:1], [int(lens[0])], D ** -0.5, [[int(lens[0]) - 1]])
    _near(out[:1, :G], want, _attention_bound(size, big, want, D, longest, dtype))


def test_decode_scale_out_and_strided_caches(ops, device):
    """A layer's caches as a slice of one pool with heads of another order, a scale of either sign, out=."""
    rng = np.random.default_rng(8)
    lens, Hq, Hkv, D, BS = [100, 23], 8, 4, 64, 32
    kc, vc, tables = _cache(rng, lens, Hkv, D, BS)
    pool = torch.zeros((Hkv, 3, 2) + kc.shape[:1] + kc.shape[2:], dtype=torch.uint8, device=device)   # [H, layer, K/V, NB, tiles, bytes]
    pool[:, 1, 0] = torch.from_numpy(kc).cuda().transpose(0, 1)
    pool[:, 1, 1] = torch.from_numpy(vc).cuda().transpose(0, 1)
    k, v = pool[:, 1, 0].transpose(0, 1), pool[:, 1, 1].transpose(0, 1)
    q, qv = _cast(rng.standard_normal((2, Hq, D)), torch.bfloat16)
    for scale in (0.3, -0.2, 0.0):
        want, size, big = _attend_all([qv[i:i + 1] for i in range(2)], kc, vc, tables, lens, scale, [[n - 1] for n in lens])
        out = torch.full((2, Hq, D), math.nan, dtype=torch.bfloat16, device=device)
        got = ops.paged_decode_kv4(q, k, v, torch.from_numpy(tables).cuda(),
                                   torch.tensor(lens, dtype=torch.int32, device=device), 100, scale=scale, out=out)
        assert got is out
        _near(out, want, _attention_bound(size, big, want, D, 100, torch.bfloat16))


def test_decode_nan_stays_in_its_head_and_large_scores(ops, device):
    rng = np.random.default_rng(4)
    lens, Hq, Hkv, D, BS = [77], 8, 8, 64, 16
    kc, vc, tables = _cache(rng, lens, Hkv, D, BS)
    kc[tables[0, 2], 3, 0, orc.scale_place(D, 5, 0, False)] = 255          # a key of head 3, a value block of head 6
    vc[tables[0, 0], 6, 0, orc.scale_place(D, 1, 1, True)] = 255
    q, qv = _cast(rng.standard_normal((1, Hq, D)) * 300, torch.float32)
    args = [torch.from_numpy(a).cuda() for a in (kc, vc, tables)]
    out = ops.paged_decode_kv4(q, *args, torch.tensor(lens, dtype=torch.int32, device=device), 77)
    want, size, big = _attend_all([qv], kc, vc, tables, lens, D ** -0.5, [[76]])
    nan = np.isnan(out.cpu().numpy())
    assert nan[0, 3].all() and nan[0, 6, 32:].all() and nan.sum() == D + 32
    keep = [h for h in range(Hq) if h not in (3, 6)]
    _near(out[:, keep], want[:, keep], _attention_bound(size, big, want, D, 77, torch.float32)[:, keep])


def test_attention_refusals(ops, device):
    kc, vc = (torch.zeros(ops.kv4_cache_shape(4, 2, 16, 64), dtype=torch.uint8, device=device) for _ in range(2))
    q = torch.zeros(3, 4, 64, device=device, dtype=torch.bfloat16)
    bt, ctx = torch.zeros(3, 2, dtype=torch.int32, device=device), torch.ones(3, dtype=torch.int32, device=device)
    for bad in (dict(block_tables=bt[:2]), dict(block_tables=bt.long()), dict(context_lens=ctx[:1]), dict(context_lens=ctx.long()),
                dict(q=q[..., :32].contiguous()), dict(q=q.double()), dict(out=q[:2]), dict(v_cache=vc[:3]),
                dict(k_cache=kc.transpose(0, 1))):
        with pytest.raises((TypeError, ValueError)):
            ops.paged_decode_kv4(**dict(dict(q=q, k_cache=kc, v_cache=vc, block_tables=bt, context_lens=ctx, max_context=5), **bad))
    seg = dict(seg_q_start=ctx, seg_len=ctx, seg_pos0=ctx)
    for bad in (dict(block_tables=bt[:2]), dict(seg_len=ctx.long()), dict(seg_pos0=ctx[:2]), dict(q=q.transpose(0, 1)),
                dict(out=q.float()), dict(q=q[..., :32].contiguous())):
        with pytest.raises((TypeError, ValueError)):
            ops.paged_prefill_kv4(**dict(dict(q=q, k_cache=kc, v_cache=vc, block_tables=bt, max_q_len=1, max_context=5, **seg), **bad))
    from mi355_paged._lib import Mi355Error
    with pytest.raises(Mi355Error, match='bad shape'):
        ops.paged_decode_kv4(q[:, :3].contiguous(), kc, vc, bt, ctx, 5)


# ------------------------------------------------------------------ prompt chunks
CHUNKS = [
    # Hq, Hkv, D, BS, chunk lengths, first positions
    (8, 8, 64, 16, [1, 5, 0, 40], [0, 30, 12, 0]),
    (8, 2, 128, 16, [33, 64], [100, 0]),
    (4, 4, 32, 32, [130, 3], [0, 260]),
    (7, 1, 64, 48, [50], [77]),
    (2, 2, 256, 16, [20, 17], [5, 0]),
    (32, 1, 64, 16, [9, 1], [0, 40]),
    (3, 3, 128, 64, [300], [0]),
    (8, 8, 64, 16, [2, 1], [1500, 900]),
]


@pytest.mark.parametrize('dtype', ALL)
@pytest.mark.parametrize('Hq,Hkv,D,BS,lens,pos0', CHUNKS, ids=lambda v: str(v))
def test_chunks(ops, device, dtype, Hq, Hkv, D, BS, lens, pos0):
    rng = np.random.default_rng(Hq + D + sum(lens))
    total = [n + p for n, p in zip(lens, pos0)]
    kc, vc, tables = _cache(rng, total, Hkv, D, BS)
    start, rows = [], 2                                        # rows before, between and behind the segments
    for n in lens:
        start.append(rows)
        rows += n + 1
    wide, val = _cast(rng.standard_normal((rows, (Hq + 1) * D)) * 1.5, dtype)
    q, qv = wide[:, D:].view(rows, Hq, D), val[:, D:].reshape(rows, Hq, D)
    want, size, big = _attend_all([qv[s:s + n] for s, n in zip(start, lens)], kc, vc, tables, total, D ** -0.5,
                                  [[p + j for j in range(n)] for n, p in zip(lens, pos0)])
    out = torch.full((rows, Hq, D), 7.0, dtype=dtype, device=device)
    meta = torch.tensor([start, lens, pos0], dtype=torch.int32, device=device)
    got = ops.paged_prefill_kv4(q, torch.from_numpy(kc).cuda(), torch.from_numpy(vc).cuda(), torch.from_numpy(tables).cuda(),
                                meta[0], meta[1], meta[2], max(lens), max(total), out=out)
    assert got is out
    inside = np.concatenate([np.arange(s, s + n) for s, n in zip(start, lens)])
    outside = np.setdiff1d(np.arange(rows), inside)
    assert bool((out[torch.from_numpy(outside).cuda()] == 7.0).all())
    _near(out[torch.from_numpy(inside).cuda()], want, _attention_bound(size, big, want, D, max(total), dtype))


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16])
def test_chunk_long_context_few_rows(ops, device, dtype):
    rng = np.random.default_rng(12)
    lens, pos0, Hq, Hkv, D, BS = [5, 1, 40], [7000, 0, 2500], 4, 2, 64, 16
    total = [n + p for n, p in zip(lens, pos0)]
    kc, vc, tables = _cache(rng, total, Hkv, D, BS)
    q, qv = _cast(rng.standard_normal((sum(lens), Hq, D)), dtype)
    start = [0, 5, 6]
    want, size, big = _attend_all([qv[s:s + n] for s, n in zip(start, lens)], kc, vc, tables, total, D ** -0.5,
                                  [[p + j for j in range(n)] for n, p in zip(lens, pos0)])
    args = [torch.from_numpy(a).cuda() for a in (kc, vc, tables)]
    meta = torch.tensor([start, lens, pos0], dtype=torch.int32, device=device)
    for bound in (7005, 50000):
        out = ops.paged_prefill_kv4(q, *args, meta[0], meta[1], meta[2], 40, bound)
        _near(out, want, _attention_bound(size, big, want, D, 7005, dtype))


WIDE = [
    # Hq, Hkv, D, BS, chunk lengths, first positions: enough rows for each way the kernel cuts them up
    (8, 8, 64, 16, [2048] * 8, [0] * 8),
    (8, 8, 64, 16, [300, 7, 400, 0, 220, 399, 350, 1], [0, 600, 0, 0, 90, 0, 17, 0]),
    (8, 8, 64, 16, [512, 500, 512, 512, 480, 512], [1300, 0, 1290, 1300, 1000, 1777]),
    (32, 8, 128, 16, [300, 290, 300, 300], [0, 0, 11, 0]),
    (32, 8, 128, 16, [256, 250, 256], [1600, 1607, 0]),
    (8, 8, 128, 16, [512, 100, 512, 512, 512], [0, 0, 0, 0, 0]),
    (4, 2, 256, 16, [200, 100], [700, 0]),
    (8, 8, 32, 16, [512, 510, 512, 512, 333, 512], [1300, 0, 1290, 1300, 1000, 1777]),
    (8, 8, 64, 16, [400] * 15 + [33], [0] * 16),
    (8, 2, 128, 16, [40, 90, 1], [900, 0, 1100]),
    (4, 4, 32, 32, [130, 3], [0, 1000]),
    (8, 8, 32, 16, [512] * 8, [300] * 8),
    (8, 8, 64, 32, [512, 511] * 4, [300] * 8),
    (8, 8, 32, 16, [2048] * 8, [0] * 8),
    (8, 8, 256, 16, [256, 250, 256] * 3, [0] * 9),
    (8, 8, 128, 16, [256, 250, 256] * 3, [0] * 9),
]


@pytest.mark.parametrize('dtype', ALL)
@pytest.mark.parametrize('Hq,Hkv,D,BS,lens,pos0', WIDE, ids=lambda v: str(v))
def test_many_rows(ops, device, dtype, Hq, Hkv, D, BS, lens, pos0):
    """Up to 40 queries of each chunk at random, the first and the last among them."""
    rng = np.random.default_rng(Hq + D + sum(lens))
    total = [n + p for n, p in zip(lens, pos0)]
    kc, vc, tables = _cache(rng, total, Hkv, D, BS)
    start = [int(x) for x in np.cumsum([0] + lens)[:-1]]
    q, qv = _cast(rng.standard_normal((sum(lens), Hq, D)) * 1.5, dtype)
    meta = torch.tensor([start, lens, pos0], dtype=torch.int32, device=device)
    out = ops.paged_prefill_kv4(q, *(torch.from_numpy(a).cuda() for a in (kc, vc, tables)), meta[0], meta[1], meta[2],
                                max(lens), max(total))
    pick = [sorted({j for j in (0, n - 1) if n} | set(rng.integers(0, n, n // 4 and min(n // 4, 40)).tolist())) for n in lens]
    want, size, big = _attend_all([qv[[s + j for j in p]] for s, p in zip(start, pick)], kc, vc, tables, total, D ** -0.5,
                                  [[p0 + j for j in p] for p0, p in zip(pos0, pick)])
    rows = torch.tensor([s + j for s, p in zip(start, pick) for j in p]).cuda()
    _near(out[rows], want, _attention_bound(size, big, want, D, max(total), dtype))


@pytest.mark.parametrize('ctx', [40, 3000])
def test_chunk_rows_outside_the_tensors_are_left_out(ops, device, ctx):
    rng = np.random.default_rng(2)
    Hq, Hkv, D, BS, rows = 4, 2, 64, 16, 20
    kc, vc, tables = _cache(rng, [ctx] * 4, Hkv, D, BS)
    big, qv = _cast(rng.standard_normal((rows + 12, Hq, D)), torch.bfloat16)
    out = torch.full((rows + 12, Hq, D), 7.0, dtype=torch.bfloat16, device=device)
    start, lens, pos0 = [0, 14, 25, -3], [4, 9, 5, 2], [ctx - 4, ctx - 9, 0, 0]
    meta = torch.tensor([start, lens, pos0], dtype=torch.int32, device=device)
    ops.paged_prefill_kv4(big[:rows], *(torch.from_numpy(a).cuda() for a in (kc, vc, tables)), meta[0], meta[1], meta[2], 9, ctx,
                          out=out[:rows])
    assert bool((out[4:14] == 7.0).all()) and bool((out[rows:] == 7.0).all())
    want, size, most = _attend_all([qv[:4], qv[14:20]], kc, vc, tables, [ctx] * 2, D ** -0.5,
                                   [[ctx - 4 + j for j in range(4)], [ctx - 9 + j for j in range(6)]])
    _near(out[[0, 1, 2, 3, 14, 15, 16, 17, 18, 19]], want, _attention_bound(size, most, want, D, ctx, torch.bfloat16))


@pytest.mark.parametrize('ctx', [60, 3000])
def test_chunk_queries_before_the_first_position_see_nothing(ops, device, ctx):
    """A negative first position: zeros, whatever the cached rows hold; the queries from position 0 on as ever.  A loose
    max_q_len and a segment longer than a tight one."""
    rng = np.random.default_rng(3)
    Hq, Hkv, D, BS = 4, 2, 64, 16
    kc, vc, tables = _cache(rng, [ctx, 40, 40], Hkv, D, BS)
    vc[tables[0, 0], :, 0, orc.scale_place(D, 0, 0, True)] = 255
    q, qv = _cast(rng.standard_normal((30, Hq, D)), torch.bfloat16)
    start, lens, pos0 = [0, 10, 20], [6, 10, 9], [-6, -4, 30]
    meta = torch.tensor([start, lens, pos0], dtype=torch.int32, device=device)
    args = [torch.from_numpy(a).cuda() for a in (kc, vc, tables)]
    want, size, most = _attend_all([qv[14:20], qv[20:29]], kc, vc, tables[1:], [40] * 2, D ** -0.5,
                                   [list(range(6)), [30 + j for j in range(9)]])
    bound = _attention_bound(size, most, want, D, 40, torch.bfloat16)
    for longest, rows in ((10, 9), (1 << 30, 9), (7, 7)):
        out = torch.full((30, Hq, D), 7.0, dtype=torch.bfloat16, device=device)
        ops.paged_prefill_kv4(q, *args, meta[0], meta[1], meta[2], longest, ctx, out=out)
        assert not out[:6].any() and not out[10:14].any() and bool((out[6:10] == 7.0).all())
        got = [j for j in range(14, 20) if j - 10 < longest] + list(range(20, 20 + rows))
        pick = [j - 14 for j in got]
        _near(out[got], want[pick], bound[pick])
        assert bool((out[20 + rows:] == 7.0).all())


@pytest.mark.parametrize('longest', [40, 1 << 31, (1 << 32) + 7, 1 << 62])
@pytest.mark.parametrize('bound', [300, (1 << 31) + 5, 1 << 62])
def test_loose_host_bounds(ops, device, longest, bound):
    """Bounds far beyond what the tensors hold say nothing: no rows and no positions are lost."""
    rng = np.random.default_rng(6)
    Hq, Hkv, D, BS = 4, 2, 64, 16
    kc, vc, tables = _cache(rng, [300, 90], Hkv, D, BS)
    args = [torch.from_numpy(a).cuda() for a in (kc, vc, tables)]
    q, _ = _cast(rng.standard_normal((60, Hq, D)), torch.bfloat16)
    meta = torch.tensor([[0, 40], [40, 20], [260, 70]], dtype=torch.int32, device=device)
    want = ops.paged_prefill_kv4(q, *args, meta[0], meta[1], meta[2], 40, 300)
    out = torch.full_like(want, 7.0)
    ops.paged_prefill_kv4(q, *args, meta[0], meta[1], meta[2], longest, bound, out=out)
    torch.testing.assert_close(out, want, atol=2.0 ** -6, rtol=2.0 ** -7)       # (another bound may cut the context up in another way)
    ctx = torch.tensor([300, 90], dtype=torch.int32, device=device)
    torch.testing.assert_close(ops.paged_decode_kv4(q[:2].contiguous(), *args, ctx, bound), ops.paged_decode_kv4(q[:2].contiguous(), *args, ctx, 300),
                               atol=2.0 ** -6, rtol=2.0 ** -7)


@pytest.mark.parametrize('Hq,Hkv,D,n,seqs,pos0', [
    (8, 8, 64, 90, 2, 0), (8, 8, 64, 512, 8, 300), (8, 8, 64, 400, 16, 0), (8, 8, 64, 2048, 8, 0), (32, 8, 128, 300, 1, 40),
    (32, 8, 128, 256, 3, 1600), (8, 2, 128, 60, 2, 1000), (8, 8, 128, 250, 9, 0), (32, 8, 128, 300, 4, 0), (8, 8, 256, 250, 9, 0), (8, 2, 256, 60, 1, 9),
    (8, 8, 32, 512, 8, 300), (8, 8, 32, 400, 16, 0), (8, 8, 32, 2048, 8, 0), (4, 2, 32, 50, 1, 5)])
def test_chunk_nan_pattern_in_every_form(ops, device, Hq, Hkv, D, n, seqs, pos0):
    """NaN value blocks within a chunk, one behind it and a NaN key: the queries that see them and no others, in the dims
    of their blocks, whichever way the kernel cuts the rows up."""
    rng = np.random.default_rng(n + D)
    G, total, BS = Hq // Hkv, n + pos0, 16
    blocks = -(-total // BS) + 1
    tables = rng.permutation(seqs * blocks).reshape(seqs, blocks).astype(np.int32)
    shape = ops.kv4_cache_shape(seqs * blocks, Hkv, BS, D)
    kc = rng.integers(0, 256, shape).astype(np.uint8)
    vc = rng.integers(0, 256, shape).astype(np.uint8)
    kc[..., 8 * D:], vc[..., 8 * D:] = 127, 127
    expect = np.zeros((seqs, n, Hq, D), dtype=bool)
    for at, head, b in ((pos0 + n // 2, Hkv - 1, 0), (pos0 + n // 2 + 1, 0, D // 32 - 1), (pos0 + n - 1, 1, D // 32 // 2), (total, 0, 0)):
        vc[tables[-1, at // BS], head, 0, orc.scale_place(D, at % 16, b, True)] = 255
        if at < total:
            expect[-1, at - pos0:, head * G:(head + 1) * G, 32 * b:32 * b + 32] = True
    at = pos0 + n // 3
    kc[tables[0, at // BS], Hkv // 2, 0, orc.scale_place(D, at % 16, 0, False)] = 255
    expect[0, at - pos0:, Hkv // 2 * G:(Hkv // 2 + 1) * G] = True
    q = torch.from_numpy(rng.standard_normal((seqs * n, Hq, D))).cuda().to(torch.bfloat16)
    meta = torch.tensor([[i * n for i in range(seqs)], [n] * seqs, [pos0] * seqs], dtype=torch.int32, device=device)
    out = ops.paged_prefill_kv4(q, torch.from_numpy(kc).cuda(), torch.from_numpy(vc).cuda(), torch.from_numpy(tables).cuda(),
                                meta[0], meta[1], meta[2], n, total)
    np.testing.assert_array_equal(torch.isnan(out).cpu().numpy().reshape(expect.shape), expect)


def test_outputs_that_overlap_their_rows_are_refused(ops, device):
    from mi355_paged._lib import Mi355Error
    qkv = torch.randn(1, 3 * 4 * 64, device=device, dtype=torch.bfloat16)
    q, k, v = (t.view(1, 4, 64) for t in qkv.chunk(3, -1))            # one token: views that are contiguous
    cos, sin = torch.ones(1, 32, device=device), torch.zeros(1, 32, device=device)
    caches = [torch.zeros(ops.kv4_cache_shape(2, 4, 16, 64), dtype=torch.uint8, device=device) for _ in range(2)]
    slots = torch.zeros(1, dtype=torch.int64, device=device)
    for x in (q, k, v):
        with pytest.raises(Mi355Error, match='overlaps'):
            ops.rope_kv4_write(q, k, v, cos, sin, slots, *caches, out=x)
    with pytest.raises(Mi355Error, match='overlaps'):
        ops.rope_rotate(q, cos, sin, out=q)


def test_chunk_nan_reaches_only_the_queries_that_see_it(ops, device):
    """A NaN key or value at a position of the chunk itself: the queries before it stay finite, whatever
    else shares their tiles."""
    rng = np.random.default_rng(5)
    n, p0, Hq, Hkv, D, BS = 45, 10, 4, 2, 64, 16
    kc, vc, tables = _cache(rng, [n + p0], Hkv, D, BS)
    q, qv = _cast(rng.standard_normal((n, Hq, D)), torch.float32)
    at = 36
    vc[tables[0, at // BS], 1, 0, orc.scale_place(D, at % 16, 0, True)] = 255       # dims 0..31 of head 1
    kc[tables[0, 50 // BS], 0, 0, orc.scale_place(D, 50 % 16, 1, False)] = 255       # a key of head 0, position 50
    args = [torch.from_numpy(a).cuda() for a in (kc, vc, tables)]
    meta = torch.tensor([[0], [n], [p0]], dtype=torch.int32, device=device)
    out = ops.paged_prefill_kv4(q, *args, meta[0], meta[1], meta[2], n, n + p0)
    want, size, big = _attend_all([qv], kc, vc, tables, [n + p0], D ** -0.5, [[p0 + j for j in range(n)]])
    nan = np.isnan(out.cpu().numpy())
    expect = np.zeros(nan.shape, dtype=bool)
    expect[at - p0:, 2:, :32] = True
    expect[50 - p0:, :2] = True
    np.testing.assert_array_equal(nan, expect)
    bound = _attention_bound(size, big, want, D, n + p0, torch.float32)
    _near(torch.where(torch.isnan(out), torch.zeros_like(out), out), np.where(expect, 0.0, want), np.where(expect, 1.0, bound))


# ------------------------------------------------------------------ slots nobody wrote
def _unwritten(rng_seed, lens, Hkv, D, BS):
    """A cache as _cache makes it, and which of its bytes belong to rows nobody wrote."""
    kc, vc, tables = _cache(np.random.default_rng(rng_seed), lens, Hkv, D, BS, fill=255)
    k0, v0, _ = _cache(np.random.default_rng(rng_seed), lens, Hkv, D, BS, fill=0)
    return kc, vc, tables, kc != k0, vc != v0


@pytest.mark.parametrize('dtype', ALL)
@pytest.mark.parametrize('Hq,Hkv,D,BS,lens,pos0', [
    (32, 8, 128, 16, [300, 290, 300, 300], [0, 0, 11, 0]), (8, 8, 64, 16, [2047, 2040] * 4, [0] * 8),
    (8, 8, 32, 16, [2047, 2041] * 4, [0] * 8), (8, 8, 256, 16, [250, 249, 251] * 3, [0] * 9), (8, 8, 64, 16, [400] * 15 + [33], [0] * 16),
    (8, 8, 64, 32, [512, 511] * 4, [301] * 8), (32, 8, 128, 16, [256, 250, 256], [1601, 1607, 0]), (4, 2, 32, 48, [7, 1], [90, 3]),
    (4, 2, 64, 16, [5, 40], [7000, 2500])], ids=lambda v: str(v)[:40])
def test_chunks_do_not_depend_on_unwritten_slots(ops, device, dtype, Hq, Hkv, D, BS, lens, pos0):
    """Contexts that end inside a tile, behind it every kind of scale byte: 0, the two that no append writes and whose
    values pass the largest bf16 (253, 254), NaN."""
    total = [n + p for n, p in zip(lens, pos0)]
    kc, vc, tables, free_k, free_v = _unwritten(sum(lens) + D, total, Hkv, D, BS)
    tables = torch.from_numpy(np.minimum(tables, len(kc) - 1)).cuda()
    q, _ = _cast(np.random.default_rng(1).standard_normal((sum(lens), Hq, D)), dtype)
    meta = torch.tensor([np.cumsum([0] + lens)[:-1].tolist(), lens, pos0], dtype=torch.int32, device=device)
    want = None
    for fill in (0, 253, 254, 255):
        kc[free_k], vc[free_v] = fill, fill
        out = ops.paged_prefill_kv4(q, torch.from_numpy(kc).cuda(), torch.from_numpy(vc).cuda(), tables, meta[0], meta[1], meta[2],
                                    max(lens), max(total))
        want = out if want is None else want
        assert torch.isfinite(out).all() and torch.equal(out, want), fill


@pytest.mark.parametrize('dtype', ALL)
@pytest.mark.parametrize('Hq,Hkv,D,BS,lens', [(8, 8, 64, 16, [1, 15, 18, 333]), (32, 8, 128, 16, [257, 50]), (4, 4, 32, 32, [5, 700, 41]),
                                              (8, 4, 256, 16, [20, 77]), (4, 2, 64, 48, [9001, 130])], ids=lambda v: str(v)[:40])
def test_decode_does_not_depend_on_unwritten_slots(ops, device, dtype, Hq, Hkv, D, BS, lens):
    kc, vc, tables, free_k, free_v = _unwritten(sum(lens) + D, lens, Hkv, D, BS)
    tables = torch.from_numpy(np.minimum(tables, len(kc) - 1)).cuda()
    q, _ = _cast(np.random.default_rng(1).standard_normal((len(lens), Hq, D)), dtype)
    want = None
    for fill in (0, 253, 254, 255):
        kc[free_k], vc[free_v] = fill, fill
        out = ops.paged_decode_kv4(q, torch.from_numpy(kc).cuda(), torch.from_numpy(vc).cuda(), tables,
                                   torch.tensor(lens, dtype=torch.int32, device=device), max(lens))
        want = out if want is None else want
        assert torch.isfinite(out).all() and torch.equal(out, want), fill


@pytest.mark.parametrize('dtype', ALL)
@pytest.mark.parametrize('byte', [253, 254])
@pytest.mark.parametrize('seqs,n,Hq,Hkv,D,pos0', [
    (1, 90, 8, 8, 64, 0), (8, 512, 8, 8, 64, 300), (16, 400, 8, 8, 64, 0), (8, 2048, 8, 8, 64, 0), (4, 300, 32, 8, 128, 0), (2, 60, 8, 2, 128, 1000),
    (9, 250, 8, 8, 256, 0), (8, 512, 8, 8, 32, 300), (8, 2048, 8, 8, 32, 0), (1, 20, 8, 2, 64, 5000)], ids=str)
def test_rows_beyond_the_format_reach_only_the_queries_that_see_them(ops, device, dtype, byte, seqs, n, Hq, Hkv, D, pos0):
    """A slot in the middle of a chunk that nobody wrote: the queries before it are what they are without it."""
    rng = np.random.default_rng(n + D)
    blocks = -(-(n + pos0) // 16)
    shape = ops.kv4_cache_shape(seqs * blocks, Hkv, 16, D)
    kc, vc = (torch.from_numpy(rng.integers(0, 256, shape, dtype=np.uint8)).cuda() for _ in range(2))
    kc[..., 8 * D:], vc[..., 8 * D:] = 126, 127
    tables = torch.arange(seqs * blocks, dtype=torch.int32, device=device).view(seqs, blocks)
    q = torch.from_numpy(rng.standard_normal((seqs * n, Hq, D))).cuda().to(dtype)
    meta = torch.tensor([[i * n for i in range(seqs)], [n] * seqs, [pos0] * seqs], dtype=torch.int32, device=device)
    args = (tables, meta[0], meta[1], meta[2], n, n + pos0)
    want = ops.paged_prefill_kv4(q, kc, vc, *args)
    at = [pos0 + n // 2, pos0 + n - 1]
    for t in at:
        for b in range(D // 32):
            vc[tables[-1, t // 16].long(), :, 0, orc.scale_place(D, t % 16, b, True)] = byte
    got = ops.paged_prefill_kv4(q, kc, vc, *args)
    before = (seqs - 1) * n + n // 2
    assert torch.isfinite(want).all() and torch.equal(got[:before], want[:before])


# ------------------------------------------------------------------ the weights' bits
def _close_bound(size, big, want, D, n, dtype):
    """_attention_bound with the 16 bits that a weight has at least: two pieces leave out 2^-16 of it, and as much may be
    missing from the sum of weights."""
    return (2 * (3 * D + 8) * U * big + 2.0 ** -22 + 2 * (n + 8) * U + 2.0 ** -15) * size + \
        (HALF[dtype] + 2 * (n + 8) * U) * np.abs(want) + 1e-30


@pytest.mark.parametrize('dtype', ALL)
@pytest.mark.parametrize('Hq,Hkv,D,lens', [(8, 8, 64, [37, 700]), (32, 8, 128, [300]), (4, 4, 32, [90, 1025]), (8, 4, 256, [50]), (4, 2, 64, [5000])],
                         ids=lambda v: str(v))
def test_decode_rounds_the_result_not_the_weights(ops, device, dtype, Hq, Hkv, D, lens):
    rng = np.random.default_rng(D + sum(lens))
    kc, vc, tables = _cache(rng, lens, Hkv, D, 16)
    B = len(lens)
    q, qv = _cast(rng.standard_normal((B, Hq, D)), dtype)
    want, size, big = _attend_all([qv[i:i + 1] for i in range(B)], kc, vc, tables, lens, D ** -0.5, [[n - 1] for n in lens])
    out = ops.paged_decode_kv4(q, torch.from_numpy(kc).cuda(), torch.from_numpy(vc).cuda(), torch.from_numpy(tables).cuda(),
                               torch.tensor(lens, dtype=torch.int32, device=device), max(lens))
    _near(out, want, _close_bound(size, big, want, D, max(lens), dtype))


@pytest.mark.parametrize('dtype', ALL)
@pytest.mark.parametrize('Hq,Hkv,D,lens,pos0', [
    (8, 8, 64, [3, 45], [0, 700]), (32, 8, 128, [300, 290, 300, 300], [0, 0, 11, 0]), (8, 8, 64, [2047, 2040] * 4, [0] * 8),
    (8, 8, 64, [512, 500, 512, 512, 480, 512], [1300, 0, 1290, 1300, 1000, 1777]), (8, 8, 256, [250, 249, 251] * 3, [0] * 9),
    (4, 4, 32, [130, 3], [0, 1000]), (8, 8, 128, [256, 250, 256] * 3, [0] * 9)], ids=lambda v: str(v)[:40])
def test_chunks_round_the_result_not_the_weights(ops, device, dtype, Hq, Hkv, D, lens, pos0):
    rng = np.random.default_rng(D + sum(lens))
    total = [n + p for n, p in zip(lens, pos0)]
    kc, vc, tables = _cache(rng, total, Hkv, D, 16)
    start = [int(x) for x in np.cumsum([0] + lens)[:-1]]
    q, qv = _cast(rng.standard_normal((sum(lens), Hq, D)), dtype)
    meta = torch.tensor([start, lens, pos0], dtype=torch.int32, device=device)
    out = ops.paged_prefill_kv4(q, *(torch.from_numpy(a).cuda() for a in (kc, vc, tables)), meta[0], meta[1], meta[2],
                                max(lens), max(total))
    pick = [sorted({0, n - 1} | set(rng.integers(0, n, min(n // 4, 12)).tolist())) for n in lens]
    want, size, big = _attend_all([qv[[s + j for j in p]] for s, p in zip(start, pick)], kc, vc, tables, total, D ** -0.5,
                                  [[p0 + j for j in p] for p0, p in zip(pos0, pick)])
    rows = torch.tensor([s + j for s, p in zip(start, pick) for j in p]).cuda()
    _near(out[rows], want, _close_bound(size, big, want, D, max(total), dtype))


@pytest.mark.parametrize('dtype', ALL)
@pytest.mark.parametrize('seqs,n,Hq,Hkv,D', [(2, 0, 8, 8, 64), (2, 0, 32, 8, 128), (1, 40, 8, 8, 64), (8, 1024, 8, 8, 64), (4, 512, 32, 8, 128),
                                             (9, 250, 8, 8, 256)])
def test_equal_value_rows_come_back(ops, device, dtype, seqs, n, Hq, Hkv, D):
    """All value rows 1.5, scores of 2^-6 q0 up to one token's 2^6 q0, far behind the others: its weight has all its bits and
    stands beside a maximum of an earlier token.  1.5 (1 +- 2^-12) rounds to 1.5 in 8 and in 11 bits; in fp32 the numerator
    and the sum of weights are sums of n terms of one sign, each off by at most n u of itself, and their quotient by one
    rounding more: 1.5 * 2 (n + 8) u = 1.9e-4 for n = 1024 (2^-15 of the weights and these stay below 2^-12)."""
    rng = np.random.default_rng(n + D)
    ctx = max(n, 600)
    code = np.full((seqs, Hkv, -(-ctx // 16), 16, D), 3, dtype=np.uint8)                 # 1.5
    byte = np.full(code.shape[:-1] + (D // 32,), 127, dtype=np.uint8)
    vc = orc.pack(code, byte, True).reshape(-1, 1, 17 * D // 2)
    code[...] = 0
    code[..., 0] = 15                                                                    # -6
    code[:, :, 0, :, 0], code[:, :, 18, 9, 0] = 0, 7                                     # the first tile 0, position 297: 6
    kc = orc.pack(code, byte, False).reshape(-1, 1, 17 * D // 2)
    blocks = -(-ctx // 16)
    kc, vc = (torch.from_numpy(np.ascontiguousarray(a.reshape(seqs, Hkv, blocks, -1).transpose(0, 2, 1, 3)).reshape(seqs * blocks, Hkv, 1, -1)).cuda()
              for a in (kc, vc))
    tables = torch.arange(seqs * blocks, dtype=torch.int32, device=device).view(seqs, blocks)
    rows = seqs * max(n, 1)
    x = np.zeros((rows, Hq, D))
    x[..., 0] = rng.uniform(0.2, 1.3, (rows, Hq))
    q, _ = _cast(x, dtype)
    if n == 0:
        out = ops.paged_decode_kv4(q, kc, vc, tables, torch.full((seqs,), ctx, dtype=torch.int32, device=device), ctx, scale=math.log(2.0))
    else:
        meta = torch.tensor([[i * n for i in range(seqs)], [n] * seqs, [ctx - n] * seqs], dtype=torch.int32, device=device)
        out = ops.paged_prefill_kv4(q, kc, vc, tables, meta[0], meta[1], meta[2], n, ctx, scale=math.log(2.0))
    _near(out, np.full(x.shape, 1.5), 1.5 * 2 * (ctx + 8) * U if dtype == torch.float32 else 0.0)


# ------------------------------------------------------------------ contexts split over workgroups
def _border_caches(rng, seqs, ctx, Hkv, D, marked):
    """Caches of sequences of ctx tokens in scattered blocks: random values; dim 0 of a key is 6 at the marked positions and
    -6 elsewhere, all else 0.  Returns (K, V, tables, values [seqs, ctx, Hkv, D])."""
    blocks = -(-ctx // 16)
    tables = rng.permutation(seqs * blocks).reshape(seqs, blocks).astype(np.int32)
    byte = np.full((seqs * blocks, Hkv, 16, D // 32), 127, dtype=np.uint8)
    kcode = np.zeros((seqs * blocks, Hkv, 16, D), dtype=np.uint8)
    flag = np.zeros(blocks * 16, dtype=bool)
    flag[marked] = True
    for i in range(seqs):
        kcode[tables[i], :, :, 0] = np.where(flag, 7, 15).reshape(blocks, 1, 16)
    vcode = rng.integers(0, 16, kcode.shape).astype(np.uint8)
    values = orc.dequantise(vcode, byte)[tables].transpose(0, 1, 3, 2, 4).reshape(seqs, blocks * 16, Hkv, D)
    return orc.pack(kcode, byte, False)[:, :, None], orc.pack(vcode, byte, True)[:, :, None], tables, values


def _border_want(values, marked, limits, G):
    """Mean of the marked value rows up to each limit, and of their magnitudes: [len(limits), Hkv * G, D]."""
    seen = [[t for t in marked if t <= lim] for lim in limits]
    return (np.repeat(np.stack([values[t].mean(0) for t in seen]), G, 1), np.repeat(np.stack([np.abs(values[t]).mean(0) for t in seen]), G, 1))


@pytest.mark.parametrize('dtype', ALL)
@pytest.mark.parametrize('B,Hq,Hkv,D,ctx,splits', [
    (16, 4, 4, 256, 2000, 4), (2, 4, 2, 256, 5000, 20), (4, 8, 8, 32, 4000, 16), (16, 8, 8, 32, 2500, 4), (3, 8, 2, 128, 3000, 12), (12, 8, 8, 128, 2000, 6),
    (2, 8, 8, 64, 6000, 24), (10, 16, 8, 64, 1500, 6)])
def test_decode_splits_lose_and_double_no_token(ops, device, dtype, B, Hq, Hkv, D, ctx, splits):
    """The tokens on either side of every border that a split may have, and a context's last, share all of the weight; one
    missing or counted twice moves every output by its value's share.  Contexts that end in front of, on and behind borders."""
    from mi355_paged import _lib
    bytes_ = _lib.load().mi355_paged_decode_kv4_workspace_bytes(B, Hq, Hkv, D, ctx, ops.dtype_code(torch.empty(0, dtype=dtype)))
    assert bytes_ == B * Hq * splits * (D + 4) * 4          # (the way of cutting up that this test is for)
    rng = np.random.default_rng(ctx + D)
    lens = [ctx] + [max(1, ctx - 127 * i - i % 3) for i in range(1, B - 1)] + [1]
    lens[1:2] = [ctx - ctx % 128]
    marked = sorted({t for t in range(ctx) if t % 128 in (0, 127)} | {n - 1 for n in lens})
    kc, vc, tables, values = _border_caches(rng, B, ctx, Hkv, D, marked)
    q = torch.zeros(B, Hq, D, dtype=dtype, device=device)
    q[..., 0] = 1.0
    args = [torch.from_numpy(a).cuda() for a in (kc, vc, tables)]
    out = ops.paged_decode_kv4(q, *args, torch.tensor(lens, dtype=torch.int32, device=device), ctx, scale=8.0)
    want, size = (np.concatenate(x) for x in zip(*[_border_want(values[i], marked, [lens[i] - 1], Hq // Hkv) for i in range(B)]))
    _near(out, want, HALF[dtype] * np.abs(want) + (2.0 ** -15 + 2 * (ctx + 8) * U) * size)
    # a NaN value block in a late split: its dims, its head's queries, the sequences that reach it
    at, head, b = ctx - 200, Hkv - 1, D // 32 - 1
    args[1][torch.from_numpy(tables[:, at // 16]).long().cuda(), head, 0, orc.scale_place(D, at % 16, b, True)] = 255
    out = ops.paged_decode_kv4(q, *args, torch.tensor(lens, dtype=torch.int32, device=device), ctx, scale=8.0)
    expect = np.zeros(want.shape, dtype=bool)
    expect[np.array(lens) > at, head * (Hq // Hkv):, 32 * b:] = True
    np.testing.assert_array_equal(torch.isnan(out).cpu().numpy(), expect)


@pytest.mark.parametrize('dtype', ALL)
@pytest.mark.parametrize('seqs,n,Hq,Hkv,D,ctx,splits', [
    (1, 16, 32, 8, 128, 4000, 16), (4, 16, 8, 8, 128, 3000, 6), (2, 16, 8, 2, 256, 3000, 12), (8, 30, 8, 8, 256, 2500, 4), (1, 9, 8, 8, 32, 5000, 20),
    (4, 20, 8, 8, 32, 2300, 5), (2, 5, 4, 2, 64, 7000, 28), (3, 40, 8, 4, 64, 2600, 6)])
def test_chunk_splits_lose_and_double_no_token(ops, device, dtype, seqs, n, Hq, Hkv, D, ctx, splits):
    from mi355_paged import _lib
    bytes_ = _lib.load().mi355_paged_prefill_kv4_workspace_bytes(seqs, seqs * n, n, Hq, Hkv, D, ctx, ops.dtype_code(torch.empty(0, dtype=dtype)))
    assert bytes_ == seqs * n * Hq * splits * (D + 4) * 4
    rng = np.random.default_rng(ctx + D)
    end = [ctx, ctx - ctx % 256 + n // 2, 256 + n // 3, n][:seqs] + [ctx - 300 * i for i in range(1, seqs - 3)]       # chunks across borders
    marked = sorted({t for t in range(ctx) if t % 128 in (0, 127)} | {t for e in end for t in range(e - n, e)})
    kc, vc, tables, values = _border_caches(rng, seqs, ctx, Hkv, D, marked)
    q = torch.zeros(seqs * n, Hq, D, dtype=dtype, device=device)
    q[..., 0] = 1.0
    args = [torch.from_numpy(a).cuda() for a in (kc, vc, tables)]
    meta = torch.tensor([[i * n for i in range(seqs)], [n] * seqs, [e - n for e in end]], dtype=torch.int32, device=device)
    out = ops.paged_prefill_kv4(q, *args, meta[0], meta[1], meta[2], n, ctx, scale=8.0)
    want, size = (np.concatenate(x) for x in zip(*[_border_want(values[i], marked, list(range(e - n, e)), Hq // Hkv) for i, e in enumerate(end)]))
    _near(out, want, HALF[dtype] * np.abs(want) + (2.0 ** -15 + 2 * (ctx + 8) * U) * size)
    # NaN value blocks in a late split: one that all queries of the first chunk see, one in the middle of the chunk
    expect = np.zeros(want.shape, dtype=bool)
    for at, head, b in ((ctx - 3 * n, 0, 0), (ctx - n // 2, Hkv - 1, D // 32 - 1)):
        args[1][int(tables[0, at // 16]), head, 0, orc.scale_place(D, at % 16, b, True)] = 255
        expect[max(0, at - (ctx - n)):n, head * (Hq // Hkv):(head + 1) * (Hq // Hkv), 32 * b:32 * b + 32] = True
    out = ops.paged_prefill_kv4(q, *args, meta[0], meta[1], meta[2], n, ctx, scale=8.0)
    np.testing.assert_array_equal(torch.isnan(out).cpu().numpy(), expect)


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('seqs,n,Hq,Hkv,D,ctx', [(3, 0, 8, 8, 64, 600), (2, 0, 8, 2, 128, 9000), (40, 0, 40, 2, 64, 300), (2, 37, 8, 2, 64, 500), (1, 9, 8, 2, 128, 6000),
                                                 (8, 512, 8, 8, 64, 812), (8, 1024, 8, 8, 64, 1024), (4, 512, 32, 8, 128, 600), (9, 250, 8, 8, 256, 600)], ids=str)
def test_attention_in_place(ops, device, dtype, seqs, n, Hq, Hkv, D, ctx):
    """out = q: a workgroup has read its query rows before it writes them."""
    rng = np.random.default_rng(ctx + D)
    blocks = -(-ctx // 16)
    kc, vc = (torch.from_numpy(rng.integers(0, 256, ops.kv4_cache_shape(seqs * blocks, Hkv, 16, D), dtype=np.uint8)).cuda() for _ in range(2))
    kc[..., 8 * D:], vc[..., 8 * D:] = 126, 127
    tables = torch.arange(seqs * blocks, dtype=torch.int32, device=device).view(seqs, blocks)
    q = torch.from_numpy(rng.standard_normal((seqs * max(n, 1), Hq, D))).cuda().to(dtype)
    if n == 0:
        lens = torch.full((seqs,), ctx, dtype=torch.int32, device=device)
        call = lambda **kw: ops.paged_decode_kv4(q, kc, vc, tables, lens, ctx, **kw)
    else:
        meta = torch.tensor([[i * n for i in range(seqs)], [n] * seqs, [ctx - n] * seqs], dtype=torch.int32, device=device)
        call = lambda **kw: ops.paged_prefill_kv4(q, kc, vc, tables, meta[0], meta[1], meta[2], n, ctx, **kw)
    want = call()
    assert call(out=q) is q and torch.equal(q, want)


# ------------------------------------------------------------------ extremes of scores and values
FORMS = [   # sequences, query rows each (0: decode), Hq, Hkv, D, context: each way rows and contexts are cut up
    (3, 0, 8, 8, 64, 600), (2, 0, 8, 2, 128, 9000), (70, 0, 8, 8, 64, 700), (1, 40, 8, 8, 64, 600), (1, 9, 8, 2, 128, 6000), (8, 512, 8, 8, 64, 812),
    (8, 1024, 8, 8, 64, 1024), (4, 512, 32, 8, 128, 600), (9, 250, 8, 8, 256, 600)]


def _attend_form(ops, form, dtype, key, value, scale):
    """Output [sequences, rows, Hq, D] (float64) of queries of ones whose cached rows have the values key(t) in their dim 0
    and value(t) in all dims; codes and scale bytes given as (code, byte) arrays over the positions."""
    seqs, n, Hq, Hkv, D, ctx = form
    blocks = -(-ctx // 16)
    caches = []
    for (code, byte), dims, last in ((key, 1, False), (value, D, True)):
        c, b = np.zeros((blocks * 16, D), dtype=np.uint8), np.full((blocks * 16, D // 32), 127, dtype=np.uint8)
        c[:ctx, :dims], b[:ctx] = code[:, None], byte[:, None]
        rec = orc.pack(c.reshape(blocks, 16, D), b.reshape(blocks, 16, D // 32), last)
        caches.append(torch.from_numpy(rec).cuda()[:, None, None].expand(-1, Hkv, 1, -1).contiguous())
    order = torch.from_numpy(np.stack([np.arange(blocks)] * seqs).astype(np.int32)).cuda()
    rows = seqs * max(n, 1)
    q = torch.zeros((rows, Hq, D), dtype=dtype, device='cuda')
    q[..., 0] = 1.0
    if n == 0:
        out = ops.paged_decode_kv4(q, *caches, order, torch.full((seqs,), ctx, dtype=torch.int32, device='cuda'), ctx, scale=scale)
    else:
        meta = torch.tensor([[i * n for i in range(seqs)], [n] * seqs, [ctx - n] * seqs], dtype=torch.int32, device='cuda')
        out = ops.paged_prefill_kv4(q, *caches, order, meta[0], meta[1], meta[2], n, ctx, scale=scale)
    return out.double().cpu().numpy().reshape(seqs, max(n, 1), Hq, D)


@pytest.mark.parametrize('dtype', ALL)
@pytest.mark.parametrize('form', FORMS, ids=str)
@pytest.mark.parametrize('scale', [1e9, 3e11, -3e11])
def test_scores_far_beyond_the_range_of_an_exponential(ops, device, dtype, form, scale):
    """Scores of 10^9 and more, where a float's last bit is far more than one power of two: the two positions that share the
    largest one share the weight, whatever step, wave or split they are in; nothing else has any."""
    ctx = form[5]
    n = max(form[1], 1)
    key = np.full(ctx, 1 if scale > 0 else 9, dtype=np.uint8)              # 0.5 (-0.5 under a negative scale)
    key[1], key[ctx - n - 2 if ctx > n + 3 else 2] = (7, 7) if scale > 0 else (15, 15)      # 6 (-6)
    code = np.where(np.arange(ctx) % 2 == 0, 2, 4).astype(np.uint8)        # 1 and 2
    value = np.array([1.0, 2.0])[np.arange(ctx) % 2]
    out = _attend_form(ops, form, dtype, (key, np.full(ctx, 127, dtype=np.uint8)), (code, np.full(ctx, 127, dtype=np.uint8)), scale)
    top = key == key[1]
    for j in range(n):
        seen = top & (np.arange(ctx) <= ctx - n + j)
        want = value[seen].mean() if seen.any() else value[0]
        np.testing.assert_array_equal(out[:, j], want)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('form', FORMS, ids=str)
def test_values_at_the_top_of_the_format(ops, device, dtype, form):
    """Values of 6 * 2^125 under a score of almost 2^8 times the weight of the maximum before it, so that the maximum may
    stay: the weighted mean is 6 * 2^125 (1 - small) and its sums stay below the largest float."""
    ctx, n = form[5], max(form[1], 1)
    key = np.zeros(ctx, dtype=np.uint8)
    key[1:], key[ctx - n - 1 if ctx > n + 2 else 300] = 15, 7               # 0 at position 0, -6 elsewhere, 6 once
    at = int(np.argmax(key == 7))
    code = np.where(np.arange(ctx) == at, 7, 0).astype(np.uint8)
    scale = 1.3 * math.log(2.0)                                             # weights 1, 2^-7.8 and 2^7.8
    out = _attend_form(ops, form, dtype, (key, np.full(ctx, 127, dtype=np.uint8)), (code, np.full(ctx, 252, dtype=np.uint8)), scale)
    weight = 2.0 ** (1.3 * np.array([0, -6, 6]))
    for j in range(n):
        m = ctx - n + j + 1
        w = np.full(m, weight[1])
        w[0] = weight[0]
        if at < m:
            w[at] = weight[2]
        want = 6 * 2.0 ** 125 * (w[at] / w.sum() if at < m else 0.0)
        bound = want * (HALF[dtype] + 2.0 ** -15 + 2 * 8 * 200 * U + 2.0 ** -22 + 4 * (m + 8) * U)
        assert (np.abs(out[:, j] - want) <= bound).all(), (j, want, out[0, j, 0, 0])


# ------------------------------------------------------------------ every form, whatever the plan would take
@pytest.mark.parametrize('dtype', ALL)
@pytest.mark.parametrize('D', [32, 64, 128, 256])
@pytest.mark.parametrize('form', [1, 2, 11, 12])
@pytest.mark.parametrize('Hq,Hkv,BS,lens,pos0', [(4, 2, 16, [1, 37, 0, 70, 130], [0, 5, 3, 33, 0]), (3, 1, 48, [45, 2, 64], [0, 1300, 1]), (8, 8, 16, [3, 33], [61, 0])],
                         ids=lambda v: str(v))
def test_chunks_in_every_form(ops, device, dtype, D, form, Hq, Hkv, BS, lens, pos0):
    """Ragged chunks in each form of the prompt kernels (two tiles only where registers hold them): results, rows outside, rows
    nobody wrote, NaN blocks; few rows behind a long context in splits where the form has them."""
    rng = np.random.default_rng(D + sum(lens))
    total = [n + p for n, p in zip(lens, pos0)]
    kc, vc, tables, free_k, free_v = _unwritten(D + sum(lens), total, Hkv, D, BS)
    tables = np.minimum(tables, len(kc) - 1)
    start = [2 + int(x) + i for i, x in enumerate(np.cumsum([0] + lens)[:-1])]
    rows = start[-1] + lens[-1] + 1
    q, qv = _cast(rng.standard_normal((rows, Hq, D)), dtype)
    bt, meta = torch.from_numpy(tables).cuda(), torch.tensor([start, lens, pos0], dtype=torch.int32, device=device)
    inside = np.concatenate([np.arange(s, s + n) for s, n in zip(start, lens)])
    outside = np.setdiff1d(np.arange(rows), inside)

    def run():
        out = torch.full((rows, Hq, D), 7.0, dtype=dtype, device=device)
        with ops.debug_knob('MI355_KV4_CHUNK_FORM', form):
            ops.paged_prefill_kv4(q, torch.from_numpy(kc).cuda(), torch.from_numpy(vc).cuda(), bt, meta[0], meta[1], meta[2], max(lens), max(total), out=out)
        assert bool((out[torch.from_numpy(outside).cuda()] == 7.0).all())
        return out[torch.from_numpy(inside).cuda()]

    want, size, big = _attend_all([qv[s:s + n] for s, n in zip(start, lens)], kc, vc, tables, total, D ** -0.5,
                                  [[p + j for j in range(n)] for n, p in zip(lens, pos0)])
    first = run()
    _near(first, want, _close_bound(size, big, want, D, max(total), dtype))
    for fill in (0, 253, 254):
        kc[free_k], vc[free_v] = fill, fill
        assert torch.equal(run(), first), fill
    # a NaN value block in the middle of the second chunk and a NaN key at its last position
    i, n, p = 1, lens[1], pos0[1]
    at, b, G = p + n // 2, D // 32 - 1, Hq // Hkv
    vc[tables[i, at // BS], 0, at % BS // 16, orc.scale_place(D, at % 16, b, True)] = 255
    kc[tables[i, (p + n - 1) // BS], Hkv - 1, (p + n - 1) % BS // 16, orc.scale_place(D, (p + n - 1) % 16, 0, False)] = 255
    expect = np.zeros(want.shape, dtype=bool)
    row0 = sum(lens[:i])
    expect[row0 + n // 2:row0 + n, :G, 32 * b:32 * b + 32] = True
    expect[row0 + n - 1, (Hkv - 1) * G:] = True
    np.testing.assert_array_equal(torch.isnan(run()).cpu().numpy(), expect)


@pytest.mark.parametrize('dtype', ALL)
@pytest.mark.parametrize('heads', [1, 2, 4, 8])
@pytest.mark.parametrize('Hq,Hkv,D,BS,lens', [(8, 8, 32, 16, [1, 33, 0, 300]), (16, 8, 32, 16, [77, 5]), (8, 8, 64, 48, [1, 17, 200]), (16, 4, 64, 16, [50, 2500]),
                                              (8, 8, 128, 16, [31, 129]), (12, 2, 128, 16, [90]), (4, 4, 256, 16, [40, 7])], ids=lambda v: str(v))
def test_decode_with_every_number_of_heads_per_wave(ops, device, dtype, heads, Hq, Hkv, D, BS, lens):
    rng = np.random.default_rng(D + sum(lens))
    kc, vc, tables, free_k, free_v = _unwritten(D + sum(lens), lens, Hkv, D, BS)
    tables = np.minimum(tables, len(kc) - 1)
    q, qv = _cast(rng.standard_normal((len(lens), Hq, D)), dtype)
    want, size, big = _attend_all([qv[i:i + 1] for i in range(len(lens))], kc, vc, tables, lens, D ** -0.5, [[n - 1] for n in lens])

    def run():
        with ops.debug_knob('MI355_KV4_DECODE_HEADS', heads):
            return ops.paged_decode_kv4(q, torch.from_numpy(kc).cuda(), torch.from_numpy(vc).cuda(), torch.from_numpy(tables).cuda(),
                                        torch.tensor(lens, dtype=torch.int32, device=device), max(lens))

    first = run()
    _near(first, want, _close_bound(size, big, want, D, max(lens), dtype))
    for fill in (0, 253, 254):
        kc[free_k], vc[free_v] = fill, fill
        assert torch.equal(run(), first), fill
    i, at, G = len(lens) - 1, lens[-1] // 2, Hq // Hkv
    vc[tables[i, at // BS], Hkv - 1, at % BS // 16, orc.scale_place(D, at % 16, 0, True)] = 255
    expect = np.zeros(want.shape, dtype=bool)
    expect[i, (Hkv - 1) * G:, :32] = True
    np.testing.assert_array_equal(torch.isnan(run()).cpu().numpy(), expect)


# ------------------------------------------------------------------ streams, graphs, all of them together
def _step(ops, s):
    """One layer's work on new rows: angles, rotation + append, attention."""
    cos, sin = ops.rope_angles(s['pos'], s['freq'])
    q = ops.rope_kv4_write(s['q'], s['k'], s['v'], cos, sin, s['slots'], s['kc'], s['vc'])
    if s['meta'] is None:
        return ops.paged_decode_kv4(q, s['kc'], s['vc'], s['tables'], s['ctx'], s['bound'])
    return ops.paged_prefill_kv4(q, s['kc'], s['vc'], s['tables'], s['meta'][0], s['meta'][1], s['meta'][2], s['longest'], s['bound'])


def _sequence_state(ops, rng, dtype, lens, new, Hq, Hkv, D, BS, decode):
    """Sequences that hold lens[i] tokens of which the last new[i] are about to be appended."""
    kc, vc, tables = _cache(rng, lens, Hkv, D, BS)
    pos = np.concatenate([np.arange(n - m, n) for n, m in zip(lens, new)])
    slots = np.concatenate([tables[i, np.arange(n - m, n) // BS].astype(np.int64) * BS + np.arange(n - m, n) % BS
                            for i, (n, m) in enumerate(zip(lens, new))])
    (q, k, v), vals = _rows(rng, len(pos), Hq, Hkv, D, dtype)
    freq, _ = ops.rope_frequencies(D)
    start = np.cumsum([0] + list(new))[:-1]
    meta = None if decode else torch.tensor(np.array([start, new, [n - m for n, m in zip(lens, new)]]), dtype=torch.int32).cuda()
    s = dict(q=q, k=k, v=v, pos=torch.from_numpy(pos).cuda(), slots=torch.from_numpy(slots).cuda(), freq=freq.cuda(),
             kc=torch.from_numpy(kc).cuda(), vc=torch.from_numpy(vc).cuda(), tables=torch.from_numpy(tables).cuda(),
             ctx=torch.tensor(lens, dtype=torch.int32).cuda(), bound=max(lens), meta=meta, longest=max(new))
    return s, vals, kc, vc, tables, pos, slots


def _expected(vals, kc, vc, tables, pos, slots, freq, lens, new, D, BS, dtype):
    """The step in float64: rotation with float32 angle rows, 4-bit rows written, attention of rounded queries."""
    a = pos[:, None] * freq
    cos, sin = np.cos(a).astype(np.float32).astype(np.float64), np.sin(a).astype(np.float32).astype(np.float64)
    qv, kv, vv = vals
    kc, vc = kc.copy(), vc.copy()
    for form, (cache, x) in enumerate(((kc, orc.rotate(kv, cos, sin, False)), (vc, vv))):
        code, byte = orc.quantise(x)
        for t, slot in enumerate(slots):
            for h in range(cache.shape[1]):
                orc.write_row(cache[slot // BS, h, slot % BS // 16], slot % 16, code[t, h], byte[t, h], bool(form))
    q = torch.from_numpy(orc.rotate(qv, cos, sin, False)).to(dtype).double().numpy()
    cut = np.split(q, np.cumsum(new)[:-1])
    return _attend_all(cut, kc, vc, tables, lens, D ** -0.5, [list(range(n - m, n)) for n, m in zip(lens, new)])


@pytest.mark.parametrize('decode', [True, False])
@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
def test_a_layers_step_together(ops, device, dtype, decode):
    rng = np.random.default_rng(21)
    lens, new = [70, 1, 33, 200], [1, 1, 1, 1] if decode else [9, 1, 33, 50]
    Hq, Hkv, D, BS = 8, 4, 64, 16
    s, vals, kc, vc, tables, pos, slots = _sequence_state(ops, rng, dtype, lens, new, Hq, Hkv, D, BS, decode)
    want, size, big = _expected(vals, kc, vc, tables, pos, slots, s['freq'].cpu().numpy(), lens, new, D, BS, dtype)
    # a query off by one rounding of its dtype moves a score by HALF * big (an angle's last bit flips 4-bit codes too
    # rarely to meet one here: 2^-24 of the values lie that near a border)
    slack = 4 * HALF[dtype] * big * size
    _near(_step(ops, s), want, _attention_bound(size, big, want, D, max(lens), dtype) + slack)


@pytest.mark.parametrize('decode', [True, False])
def test_captured_and_replayed(ops, device, decode):
    """The step as a graph, replayed on new inputs between eager work of other shapes that grows the shared
    workspace, and on a stream of its own."""
    rng = np.random.default_rng(30)
    lens, new = [3000, 64, 900], [1, 1, 1] if decode else [2, 64, 20]
    mk = lambda: _sequence_state(ops, rng, torch.bfloat16, lens, new, 8, 4, 64, 16, decode)[0]
    s, fresh = mk(), [mk() for _ in range(3)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _step(ops, s)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _step(ops, s)
    big = _sequence_state(ops, rng, torch.bfloat16, [6000, 5000], [1, 1], 8, 4, 64, 16, True)[0]
    for f in fresh:
        for name in ('q', 'k', 'v', 'pos', 'slots', 'kc', 'vc', 'tables', 'ctx'):
            s[name].copy_(f[name])
        graph.replay()
        _step(ops, big)                       # eager, larger: a workspace shared with the graph would be overwritten
        got = out.clone()
        torch.cuda.synchronize()
        assert torch.equal(got, _step(ops, f))
        assert torch.equal(s['kc'], f['kc']) and torch.equal(s['vc'], f['vc'])
    with torch.cuda.stream(side):
        other = _step(ops, fresh[0])
    side.synchronize()
    assert torch.equal(other, _step(ops, fresh[0]))


@pytest.mark.parametrize('decode', [True, False])
def test_two_streams_at_once(ops, device, decode):
    """Split launches of two sizes in flight together: each stream has partial sums of its own."""
    rng = np.random.default_rng(31)
    steps = [_sequence_state(ops, rng, torch.bfloat16, lens, new, 8, 4, 64, 16, decode)[0]
             for lens, new in (([6000, 300], [1, 1] if decode else [3, 40]), ([4000, 5000, 17], [1, 1, 1] if decode else [20, 9, 17]))]
    want = [_step(ops, s) for s in steps]
    streams = [torch.cuda.Stream() for _ in steps]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for side, s, outs in zip(streams, steps, got):
            with torch.cuda.stream(side):
                outs.append(_step(ops, s))
    torch.cuda.synchronize()
    for outs, w in zip(got, want):
        assert all(torch.equal(o, w) for o in outs)


def test_blocks_far_into_a_large_pool(ops, device):
    """Records beyond 2^32 bytes: the same step over a pool of 6 GiB per tensor and over a small one."""
    rng = np.random.default_rng(32)
    Hkv, D, BS = 4, 128, 16
    lens, new = [500, 40], [70, 40]
    s = _sequence_state(ops, rng, torch.bfloat16, lens, new, 8, Hkv, D, BS, False)[0]
    far = dict(s)
    shape = ops.kv4_cache_shape((6 << 30) // (Hkv * 17 * D // 2), Hkv, BS, D)
    move = shape[0] - s['kc'].shape[0]
    for name in ('kc', 'vc'):
        far[name] = torch.empty(shape, dtype=torch.uint8, device=device)
        far[name][move:] = s[name]
    far['tables'], far['slots'] = s['tables'] + move, s['slots'] + move * BS
    assert move * Hkv * 17 * D // 2 > 1 << 32
    assert torch.equal(_step(ops, far), _step(ops, s))
    assert torch.equal(far['kc'][move:], s['kc']) and torch.equal(far['vc'][move:], s['vc'])
    ctx = torch.tensor(lens, dtype=torch.int32, device=device)
    q = s['q'][:2].contiguous()
    assert torch.equal(ops.paged_decode_kv4(q, far['kc'], far['vc'], far['tables'], ctx, 500),
                       ops.paged_decode_kv4(q, s['kc'], s['vc'], s['tables'], ctx, 500))
    for a, b in zip(ops.kv4_read_slots(far['kc'], far['vc'], far['slots']), ops.kv4_read_slots(s['kc'], s['vc'], s['slots'])):
        assert torch.equal(a, b)


def test_blocks_of_more_than_2_to_the_31_bytes(ops, device):
    """One block that holds a whole long sequence, 2.2 GB per tensor: rows at its end are written, read and attended to.
    Keys of 0 everywhere else, whose 16 million weights are e^-70 of the last rows' at most."""
    D, tiles, n = 256, 1_000_000, 40
    ctx = tiles * 16 - 7
    shape = ops.kv4_cache_shape(1, 1, tiles * 16, D)
    assert shape[2] * shape[3] > 1 << 31
    kc, vc = (torch.full(shape, 0, dtype=torch.uint8, device=device) for _ in range(2))
    for c in (kc, vc):
        c[..., 8 * D:] = 127
    rng = np.random.default_rng(9)
    x = torch.from_numpy(rng.choice([-1.0, 1.0], (n, 3, D))).cuda().to(torch.bfloat16)
    q, k, v = x[:, :1].contiguous() * 0.5, x[:, :1].contiguous() * 3, x[:, 2:].contiguous()
    slots = torch.arange(ctx - n, ctx, device=device)
    out = ops.rope_kv4_write(q, k, v, None, None, slots, kc, vc)
    assert torch.equal(out, q)
    rk, rv = ops.kv4_read_slots(kc, vc, slots)
    assert torch.equal(rk, k) and torch.equal(rv, v)
    table, scale = torch.zeros(1, 1, dtype=torch.int32, device=device), 0.25                          # a row's own score is 96, the others' have a spread of 6
    got = ops.paged_decode_kv4(q[-1:].contiguous(), kc, vc, table, torch.tensor([ctx], dtype=torch.int32, device=device), ctx, scale=scale)
    meta = torch.tensor([[0], [n], [ctx - n]], dtype=torch.int32, device=device)
    chunk = ops.paged_prefill_kv4(q, kc, vc, table, meta[0], meta[1], meta[2], n, ctx, scale=scale)
    qd, kd, vd = (t.double()[:, 0] for t in (q, k, v))
    score = qd @ kd.T * scale
    score = score.masked_fill(torch.ones_like(score).triu(1).bool(), -math.inf)
    want = (torch.softmax(score, -1) @ vd).cpu().numpy()
    bound = 2.0 ** -8 * np.abs(want) + 2.0 ** -14 + 2.0 ** -22
    _near(chunk[:, 0], want, bound)
    _near(got[:, 0], want[-1:], bound[-1:])


# ------------------------------------------------------------------ the engine over a 4-bit cache
@pytest.mark.parametrize('rotary', [None, dict(dim=32, interleaved=True, scaling={'kind': 'yarn', 'factor': 4, 'original': 64})])
def test_engine_layer_steps(ops, device, rotary):
    """Two steps of an attention layer (prompts, then a decode token beside a later chunk) against float64 on the
    layer's own projections: which rows are rotated how, where they are cached and who attends to what."""
    import mini_vllm as mv
    torch.manual_seed(3)
    H, D, BS = 4, 64, 16
    pos_cfg = mv.RotaryPositions(D, **(rotary or {}))
    layer = mv.SelfAttention(H * D, H, D, pos_cfg).to(device)
    kc, vc = (torch.full(ops.kv4_cache_shape(8, H, BS, D), 255, dtype=torch.uint8, device=device) for _ in range(2))
    okc, ovc = kc.cpu().numpy(), vc.cpu().numpy()
    tables = [[5, 2, 0], [1, 7, 3]]
    steps = [([0, 0], [20, 17], [True, True]), ([20, 17], [1, 14], [False, True])]       # starts, lengths, prefill?
    for starts, lens, prefill in steps:
        pos = np.concatenate([np.arange(s, s + n) for s, n in zip(starts, lens)])
        slots = np.concatenate([[t[p // BS] * BS + p % BS for p in range(s, s + n)] for t, s, n in zip(tables, starts, lens)])
        plan = mv.build_attn_plan(pos.tolist(), lens, prefill, tables, device, append_ok=True, from_cache=True)
        x = torch.randn(len(pos), H * D, device=device)
        with torch.no_grad():
            got = layer(x, torch.from_numpy(pos).cuda(), (kc, vc), torch.from_numpy(slots).cuda(), lens, prefill, plan)
            qkv = layer.qkv(x).double().cpu().numpy()
        q, k, v = (t.reshape(len(pos), H, D) for t in np.split(qkv, 3, -1))
        cos, sin = (t.double().cpu().numpy() for t in pos_cfg.angles(torch.from_numpy(pos).cuda()))
        for form, (cache, rows) in enumerate(((okc, orc.rotate(k, cos, sin, pos_cfg.interleaved)), (ovc, v))):
            code, byte = orc.quantise(rows)
            for t, slot in enumerate(slots):
                for h in range(H):
                    orc.write_row(cache[slot // BS, h, slot % BS // 16], slot % 16, code[t, h], byte[t, h], bool(form))
        np.testing.assert_array_equal(kc.cpu().numpy(), okc)
        np.testing.assert_array_equal(vc.cpu().numpy(), ovc)
        rot = orc.rotate(q, cos, sin, pos_cfg.interleaved)
        total = [s + n for s, n in zip(starts, lens)]
        want, size, big = _attend_all(np.split(rot, [lens[0]]), okc, ovc, np.array(tables), total, D ** -0.5,
                                      [list(range(s, s + n)) for s, n in zip(starts, lens)])
        # per attention output: the kernel's bound and one rounding of the rotated query; then a product of H D terms
        bound = _attention_bound(size, big, want, D, max(total), torch.float32) + 8 * U * big * size
        w = layer.out_proj.weight.detach().double().cpu().numpy()
        a = want.reshape(len(pos), -1)
        _near(got, a @ w.T, bound.reshape(len(pos), -1) @ np.abs(w).T + (H * D + 2) * U * (np.abs(a) @ np.abs(w).T))


@pytest.mark.parametrize('kw', [dict(kv_cache_dtype='mxfp4'), dict(rotary=dict(dim=16))], ids=str)
def test_a_plan_serves_calls_with_other_positions(device, kw):
    """One plan object for two steps whose tensors are updated in place, and for a single layer afterwards: every call
    rotates by its own positions."""
    import mini_vllm as mv
    results = []
    for fresh in (True, False):
        torch.manual_seed(3)
        model = mv.MiniTransformer(100, 64, 2, 2, 64, 8, 16, **kw).to(device)
        ids = torch.tensor([5, 9], device=device)
        tables = torch.tensor([[1, 2], [4, 3]], dtype=torch.int32, device=device)
        ctx = torch.ones(2, dtype=torch.int32, device=device)
        mk = lambda: mv.AttnPlan(total_tokens=2, causal_index=None, cu_seqlens=None, causal_tokens=0, max_causal_len=0, paged_index=None,
                                 paged_tables=tables, paged_context=ctx, paged_rows=2, max_context=32, pure_decode=True)
        plan, outs = mk(), []
        with torch.no_grad():
            for step in range(3):
                pos = torch.full((2,), step, dtype=torch.int64, device=device)
                slots = tables[:, 0].long() * 16 + pos
                ctx.fill_(step + 1)
                outs.append(model.forward_planned(ids, pos, slots, mk() if fresh else plan))
            x = torch.randn(2, 64, generator=torch.Generator(device).manual_seed(1), device=device)
            pos = torch.full((2,), 3, dtype=torch.int64, device=device)
            ctx.fill_(4)
            outs.append(model.layers[0].attn(x, pos, (model.k_cache[0], model.v_cache[0]), tables[:, 0].long() * 16 + pos, [1, 1], [False] * 2,
                                             mk() if fresh else plan))
        results.append(outs)
    for a, b in zip(*results):
        assert torch.equal(a, b)


def _generate(mv, graphs, dtype, **kw):
    torch.manual_seed(7)
    eng = mv.MiniVLLM(vocab_size=300, hidden_size=128, num_layers=2, num_heads=4, intermediate_size=256, num_kv_blocks=64,
                      block_size=16, max_num_seqs=8, max_num_batched_tokens=64, device='cuda', dtype=dtype,
                      decode_graphs=graphs, **kw)
    rng = np.random.default_rng(1)
    for n in (5, 90, 33, 1, 130):
        eng.add_request(rng.integers(1, 300, n).tolist(), max_new_tokens=12, temperature=0.0)
    out = {}
    while eng.scheduler.has_unfinished:
        for rid, tok in eng.step():
            out.setdefault(rid, []).append(tok)
    return out, eng


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('kw', [dict(kv_cache_dtype='mxfp4'), dict(kv_cache_dtype='mxfp4', rotary=dict(dim=16, interleaved=True)),
                                dict(rotary=dict(scaling={'kind': 'linear', 'factor': 2.0}))], ids=str)
def test_engine_generates_the_same_with_and_without_graphs(device, dtype, kw):
    """Chunked prompts, mixed and pure decode steps: replayed steps give what eager ones give, to the token."""
    import mini_vllm as mv
    a, eng = _generate(mv, True, dtype, **kw)
    b, _ = _generate(mv, False, dtype, **kw)
    assert a == b and all(len(v) == 12 or v[-1] == 0 for v in a.values()) and len(a) == 5
    assert eng._launches > 0 and torch.isfinite(eng.last_logits.float()).all()
    if 'kv_cache_dtype' in kw:
        assert eng.model.k_cache.dtype == torch.uint8


def test_engine_rotary_settings_equal_the_table_where_they_mean_the_same(device):
    """rotary={} is the reference's rotation, with angles formed in double instead of taken from a float table: at
    positions below 150 an angle differs by at most 150 * 2^-24 = 9e-6, a score by a few times that, and two layers
    of this model turn it into logits within 1e-3 of each other."""
    import mini_vllm as mv
    logits = []
    for kw in ({}, dict(rotary={})):
        torch.manual_seed(7)
        model = mv.MiniTransformer(300, 128, 2, 4, 256, 16, 16, **kw).to(device)
        n = 140
        pos = torch.arange(n, device=device)
        with torch.no_grad():
            logits.append(model(torch.arange(1, n + 1, device=device), pos, pos, [n], [True], block_tables=[list(range(9))]))
    torch.testing.assert_close(logits[0], logits[1], atol=1e-3, rtol=1e-3)


def test_engine_prefix_caching_over_a_4_bit_cache(device):
    """Requests that share full prompt blocks read the 4-bit blocks of the first; tokens as without sharing (float32
    activations: weights carry 24 bits, so the way a prompt is cut moves logits by rounding only)."""
    import mini_vllm as mv
    rng = np.random.default_rng(3)
    prefix, tails = rng.integers(1, 300, 70).tolist(), [rng.integers(1, 300, n).tolist() for n in (9, 30, 1)]
    results = []
    for caching in (True, False):
        torch.manual_seed(7)
        eng = mv.MiniVLLM(vocab_size=300, hidden_size=128, num_layers=2, num_heads=4, intermediate_size=256, num_kv_blocks=40,
                          block_size=16, max_num_seqs=4, max_num_batched_tokens=48, device='cuda', dtype=torch.float32,
                          kv_cache_dtype='mxfp4', enable_prefix_caching=caching)
        out = []
        for tail in tails + tails[:1]:
            eng.add_request(prefix + tail, max_new_tokens=10, temperature=0.0)
            got = []
            while eng.scheduler.has_unfinished:
                got += [tok for _, tok in eng.step()]
            out.append(got)
        results.append(out)
    assert results[0] == results[1] and results[0][0] == results[0][3]
