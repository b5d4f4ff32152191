"""The 4-bit KV cache's operators, as cases that can be timed and compared: rotary angles from positions, rotation +
4-bit append to a paged cache, decode attention over that cache and attention of prompt chunks over it.

The plain forms below are elementary torch operations in 32 bits (64 for angles and for values next to a rounding
border).  With `own` set, `run` calls the framework's kernels instead.

The cache format.  A cache tensor is uint8 [blocks, kv_heads, block_size / 16, 17 * D / 2]: per block, head and tile of
16 tokens one record of 8 D bytes of E2M1 codes followed by D / 2 bytes of E8M0 scales (value = code value * 2^(byte - 127);
byte 255 = the block of 32 is NaN).  A scale covers 32 consecutive dims of one token's head row.
  K record: codes [16 tokens][D / 2] (even dim in the low nibble), scales [16 tokens][D / 32].
  V record: codes [4 token groups][16 dim pairs][D / 32][4 tokens]: the byte at [g][c][b][j] holds dims 32 b + 2 c (low
            nibble) and 32 b + 2 c + 1 of token 4 g + j; scales [4 token groups][D / 32][4 tokens].
"""
import math
import os
import random
import sys

import torch

own = False

_DTYPES = {'bf16': torch.bfloat16, 'fp16': torch.float16, 'fp32': torch.float32}
_MAGNITUDES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _ops():
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), 'vllm-from-scratch_amd')
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from mi355_paged import ops
    return ops


# ---------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # the angles of one small decode step; of a long prompt's chunk at positions around a million, frequencies
        # stretched for a long context
        dict(name='angles_decode', op='angles', T=64, half=32, start=2048, stretch=1.0),
        dict(name='angles_prompt', op='angles', T=16384, half=64, start=1000000, stretch=32.0),
        # a decode step's append: 256 sequences, 8 heads of 64, one token each
        dict(name='append_decode', op='append', T=256, Hq=8, Hkv=8, D=64, BS=16, rotary=64, interleaved=False,
             run=1, dtype='bf16'),
        # a prompt batch with grouped heads, interleaved rotation of half of the head
        dict(name='append_prompt', op='append', T=8192, Hq=32, Hkv=8, D=128, BS=16, rotary=64, interleaved=True,
             run=2048, dtype='bf16'),
        # an odd number of tokens in runs that end inside a tile, float32 activations
        dict(name='append_odd_fp32', op='append', T=1037, Hq=8, Hkv=8, D=32, BS=32, rotary=32, interleaved=False,
             run=61, dtype='fp32'),
        # one short sequence: latency
        dict(name='decode_one', op='decode', B=1, Hq=8, Hkv=8, D=64, BS=16, lo=37, hi=37, dtype='bf16'),
        # the headline batch of the 16-bit cache: 256 sequences of 2048 tokens, 8 heads of 64
        dict(name='decode_batch', op='decode', B=256, Hq=8, Hkv=8, D=64, BS=16, lo=2048, hi=2048, dtype='bf16'),
        # few long sequences with grouped heads, ragged, half precision
        dict(name='decode_long_gqa', op='decode', B=4, Hq=32, Hkv=8, D=128, BS=16, lo=20001, hi=65536, dtype='fp16'),
        # the small model's step: 16 ragged sequences, 8 heads of 32, float32
        dict(name='decode_small_fp32', op='decode', B=16, Hq=8, Hkv=8, D=32, BS=16, lo=1, hi=700, dtype='fp32'),
        # short chunks behind short prefixes (a mixed step of the engine)
        dict(name='chunk_short', op='chunk', n=8, Hq=8, Hkv=8, D=64, BS=16, lo=1, hi=45, plo=0, phi=900, dtype='bf16'),
        # long prompt chunks behind a prefix of the same length, grouped heads
        dict(name='chunk_long_gqa', op='chunk', n=4, Hq=32, Hkv=8, D=128, BS=16, lo=2048, hi=2048, plo=2048, phi=2048,
             dtype='bf16'),
        # whole prompts of uneven lengths, half precision
        dict(name='chunk_ragged_fp16', op='chunk', n=12, Hq=8, Hkv=8, D=64, BS=16, lo=33, hi=1500, plo=0, phi=0,
             dtype='fp16'),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(['angles', 'append', 'append', 'decode', 'decode', 'decode', 'chunk', 'chunk', 'chunk'])
    if op == 'angles':
        return dict(op=op, T=_log(rng, 1, 16384), half=8 * rng.randint(1, 16), start=_log(rng, 1, 1 << 24),
                    stretch=rng.choice([1.0, 4.0, 32.0]))
    D = rng.choice([32, 64, 64, 128, 128, 256])
    Hkv = rng.choice([1, 2, 4, 6, 8, 8])
    G = rng.choice([1, 1, 2, 4, 7, 8])
    dtype = rng.choice(['bf16', 'bf16', 'fp16', 'fp32'])
    BS = rng.choice([16, 16, 32, 64])
    c = dict(op=op, Hq=G * Hkv, Hkv=Hkv, D=D, BS=BS, dtype=dtype)
    if op == 'append':
        T = _log(rng, 1, 8192)
        return dict(c, T=T, rotary=rng.choice([r for r in (0, 16, 32, 64, 128, 256) if r <= D]),
                    interleaved=rng.random() < 0.5, run=_log(rng, 1, T))
    if op == 'decode':
        B = _log(rng, 1, 256)
        hi = _log(rng, 1, max(1, min(65536, (1 << 31) // (B * Hkv * D * 8))))
        return dict(c, B=B, lo=rng.randint(1, hi), hi=hi)
    n = _log(rng, 1, 16)
    hi = _log(rng, 1, 2048)
    phi = rng.choice([0, _log(rng, 1, 4096)])
    while n * c['Hq'] * hi * (hi + phi) > 4 * 32 * 2048 * 4096:
        n, hi = max(1, n // 2), hi if n > 1 else hi // 2
    return dict(c, n=n, lo=rng.randint(1, hi), hi=hi, plo=rng.randint(0, phi), phi=phi)


def _between(lo, hi, n, salt):
    """n lengths in [lo, hi], the last one hi; a function of the case alone."""
    r = random.Random(7919 * n + 31 * hi + lo + salt)
    return [r.randint(lo, hi) for _ in range(n - 1)] + [hi]


def _lengths(case):
    if case['op'] == 'decode':
        return _between(case['lo'], case['hi'], case['B'], 1)
    return (_between(case['lo'], case['hi'], case['n'], 2), _between(case['plo'], case['phi'], case['n'], 3))


def work(case):
    if case['op'] == 'angles':
        pairs = case['T'] * case['half']
        return dict(bytes=8 * case['T'] + 8 * case['half'] + 8 * pairs, flops=8 * pairs)
    esize = 4 if case['dtype'] == 'fp32' else 2
    Hq, Hkv, D = case['Hq'], case['Hkv'], case['D']
    row4 = Hkv * D * 17 // 32                       # one token's 4-bit K (or V) rows with their scales
    if case['op'] == 'append':
        T = case['T']
        # q in and out, k and v in, the cache rows out, the angles and slots in, the written values out
        return dict(bytes=T * (2 * Hq * D * esize + 4 * Hkv * D * esize + 2 * row4 + 4 * case['rotary'] + 8),
                    flops=T * (3 * (Hq + Hkv) * case['rotary'] + 8 * Hkv * D))
    if case['op'] == 'decode':
        lens = _lengths(case)
        return dict(bytes=sum(lens) * 2 * row4 + len(lens) * (2 * Hq * D * esize + 4)
                    + 4 * sum(-(-n // case['BS']) for n in lens), flops=4 * sum(lens) * Hq * D)
    lens, pos0 = _lengths(case)
    pairs = sum(n * p + n * (n + 1) // 2 for n, p in zip(lens, pos0))
    return dict(bytes=sum(n + p for n, p in zip(lens, pos0)) * 2 * row4 + sum(lens) * 2 * Hq * D * esize,
                flops=4 * pairs * Hq * D)


# ---------------------------------------------------------------------------------------------- inputs
def _quantise(x):
    """Codes (uint8, 0..15) and scale bytes (uint8, last dim / 32) of x [..., D]; any float type."""
    blocks = x.unflatten(-1, (-1, 32))
    a = blocks.abs()
    top = a.amax(-1, keepdim=True)
    m, e = torch.frexp(top)                         # top = m * 2^e, m in [0.5, 1)
    e = (e - 3 + (m > 0.75)).clamp(-120, 125)       # the smallest power with top <= 6 * 2^e
    e = torch.where(top > 0, e, torch.full_like(e, -120))
    t = torch.ldexp(a, -e)
    code = ((t > 0.25).to(torch.uint8) + (t >= 0.75) + (t > 1.25) + (t >= 1.75) + (t > 2.5) + (t >= 3.5) + (t > 5.0))
    code = code.to(torch.uint8) | ((blocks < 0) & (code > 0)).to(torch.uint8) << 3
    return code.flatten(-2), (e.squeeze(-1) + 127).to(torch.uint8)


def _values(code, scale):
    """Codes and scale bytes -> float32 values."""
    table = torch.tensor(_MAGNITUDES + tuple(-m for m in _MAGNITUDES), device=code.device)
    power = torch.ldexp(torch.ones((), device=code.device), scale.to(torch.int32) - 127)
    power = torch.where(scale == 255, torch.full_like(power, math.nan), power)
    return table[code.int()] * power.repeat_interleave(32, -1)


def _pack(code, scale, value_form):
    """[..., 16 tokens, D] codes and [..., 16, D / 32] scales -> records [..., 17 D / 2]."""
    byte = code[..., 0::2] | code[..., 1::2] << 4
    if value_form:                                  # [g, j, b, c] -> [g, c, b, j];  [g, j, b] -> [g, b, j]
        byte = byte.unflatten(-1, (-1, 16)).unflatten(-3, (4, 4)).transpose(-3, -1).transpose(-2, -1)
        byte = byte.transpose(-2, -1)
        byte = byte.flatten(-4, -1)
        scale = scale.unflatten(-2, (4, 4)).transpose(-2, -1).flatten(-3, -1)
    else:
        byte, scale = byte.flatten(-2, -1), scale.flatten(-2, -1)
    return torch.cat([byte, scale], -1)


def _unpack(record, value_form):
    """Records [..., 17 D / 2] -> codes [..., 16, D], scales [..., 16, D / 32]."""
    D = record.shape[-1] * 2 // 17
    byte, scale = record[..., :8 * D], record[..., 8 * D:]
    if value_form:
        byte = byte.unflatten(-1, (4, 16, D // 32, 4)).transpose(-3, -1).flatten(-2, -1).flatten(-3, -2)
        scale = scale.unflatten(-1, (4, D // 32, 4)).transpose(-2, -1).flatten(-3, -2)
    else:
        byte, scale = byte.unflatten(-1, (16, D // 2)), scale.unflatten(-1, (16, D // 32))
    return torch.stack([byte & 15, byte >> 4], -1).flatten(-2, -1), scale


def _generator(seed):
    return torch.Generator(device='cuda').manual_seed(seed)


def _cached(g, case, blocks, spread):
    """One cache tensor of random rows; `spread`: dims of their own size, as keys have."""
    D, tiles = case['D'], blocks * case['Hkv'] * case['BS'] // 16
    size = torch.exp2(spread * torch.randn(D, generator=g, device='cuda'))
    out = torch.empty(tiles, 17 * D // 2, dtype=torch.uint8, device='cuda')
    for at in range(0, tiles, 1 << 17):
        rows = torch.randn(min(1 << 17, tiles - at), 16, D, generator=g, device='cuda') * size
        out[at:at + rows.shape[0]] = _pack(*_quantise(rows), value_form=spread == 0.0)
    return out.view(blocks, case['Hkv'], case['BS'] // 16, 17 * D // 2)


def _tables(g, lens, BS):
    """Block tables of sequences that own random blocks of a pool, and the pool's size."""
    need = [-(-n // BS) for n in lens]
    blocks = sum(need) + 3
    order = torch.randperm(blocks, generator=g, device='cuda').to(torch.int32)
    wide = torch.zeros(len(lens), max(need), dtype=torch.int32)
    start = [sum(need[:i]) for i in range(len(need))]
    at = torch.cat([torch.arange(n) + s for n, s in zip(need, start)])
    row = torch.cat([torch.full((n,), i) for i, n in enumerate(need)])
    col = torch.cat([torch.arange(n) for n in need])
    wide = wide.cuda()
    wide[row.cuda(), col.cuda()] = order[at.cuda()]
    return wide, blocks


def _angles_state(case, seed):
    g = _generator(seed)
    jump = torch.randint(0, 4, (case['T'],), generator=g, device='cuda')
    i = torch.arange(case['half'], dtype=torch.float64, device='cuda')
    return dict(op='angles', positions=case['start'] + torch.cumsum(jump, 0),
                freq=10000.0 ** (-i / case['half']) / case['stretch'], factor=1.0 + 0.1 * math.log(case['stretch']))


def _append_state(case, seed):
    g = _generator(seed)
    T, Hq, Hkv, D, BS, dtype = (case['T'], case['Hq'], case['Hkv'], case['D'], case['BS'], _DTYPES[case['dtype']])
    # runs of consecutive positions, each in a sequence of its own that starts somewhere in its first tile
    runs = [min(case['run'], T - at) for at in range(0, T, case['run'])]
    r = random.Random(seed)
    first = [r.randrange(16) for _ in runs]
    tables, blocks = _tables(g, [n + f for n, f in zip(runs, first)], BS)
    start = torch.tensor(first).repeat_interleave(torch.tensor(runs))
    run_at = torch.tensor([sum(runs[:i]) for i in range(len(runs))]).repeat_interleave(torch.tensor(runs))
    pos = (start + torch.arange(T) - run_at).cuda()
    seq = torch.arange(len(runs)).repeat_interleave(torch.tensor(runs)).cuda()
    qkv = torch.randn(T, (Hq + 2 * Hkv) * D, generator=g, device='cuda').to(dtype)
    s = dict(op='append', interleaved=case['interleaved'], qkv=qkv, Hq=Hq, Hkv=Hkv, D=D,
             slots=tables[seq, pos // BS].long() * BS + pos % BS, cos=None, sin=None,
             k_cache=torch.zeros(blocks, Hkv, BS // 16, 17 * D // 2, dtype=torch.uint8, device='cuda'),
             v_cache=torch.zeros(blocks, Hkv, BS // 16, 17 * D // 2, dtype=torch.uint8, device='cuda'))
    if case['rotary']:
        half = case['rotary'] // 2
        ang = (pos + 1000).double()[:, None] * 10000.0 ** (-torch.arange(half, device='cuda').double() / half)
        s['cos'], s['sin'] = ang.cos().float(), ang.sin().float()
    return s


def _decode_state(case, seed):
    g = _generator(seed)
    lens = _lengths(case)
    tables, blocks = _tables(g, lens, case['BS'])
    q = torch.randn(len(lens), case['Hq'], case['D'], generator=g, device='cuda').to(_DTYPES[case['dtype']])
    return dict(op='decode', q=q, k_cache=_cached(g, case, blocks, 0.5), v_cache=_cached(g, case, blocks, 0.0),
                tables=tables, lens=torch.tensor(lens, dtype=torch.int32, device='cuda'), longest=max(lens))


def _chunk_state(case, seed):
    g = _generator(seed)
    lens, pos0 = _lengths(case)
    tables, blocks = _tables(g, [n + p for n, p in zip(lens, pos0)], case['BS'])
    q = torch.randn(sum(lens), case['Hq'], case['D'], generator=g, device='cuda').to(_DTYPES[case['dtype']])
    start = [sum(lens[:i]) for i in range(len(lens))]
    each = torch.tensor(lens)
    meta = torch.tensor([start, lens, pos0], dtype=torch.int32, device='cuda')
    return dict(op='chunk', q=q, k_cache=_cached(g, case, blocks, 0.5), v_cache=_cached(g, case, blocks, 0.0),
                tables=tables, meta=meta, longest=max(lens), context=max(n + p for n, p in zip(lens, pos0)),
                seg=torch.arange(len(lens)).repeat_interleave(each).cuda(),
                off=(torch.arange(sum(lens)) - torch.tensor(start).repeat_interleave(each)).cuda())


_STATES = dict(angles=_angles_state, append=_append_state, decode=_decode_state, chunk=_chunk_state)


def prepare(case, seed):
    return _STATES[case['op']](case, seed)


# ---------------------------------------------------------------------------------------------- plain forms
def _plain_angles(s):
    ang = s['positions'].double()[:, None] * s['freq']
    return dict(cos=(ang.cos() * s['factor']).float(), sin=(ang.sin() * s['factor']).float())


def _rotated(x, cos, sin, interleaved):
    """x [T, H, D] with its first 2 * half dims rotated, in the type of cos."""
    x = x.to(cos.dtype)
    R = 2 * cos.shape[1]
    c, s = cos[:, None], sin[:, None]
    if interleaved:
        a, b = x[..., 0:R:2], x[..., 1:R:2]
        turned = torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)
    else:
        a, b = x[..., :R // 2], x[..., R // 2:R]
        turned = torch.cat([a * c - b * s, b * c + a * s], -1)
    return torch.cat([turned, x[..., R:]], -1)


def _plain_append(s):
    T, Hq, Hkv, D = s['qkv'].shape[0], s['Hq'], s['Hkv'], s['D']
    q, k, v = (t.view(T, -1, D) for t in s['qkv'].split([Hq * D, Hkv * D, Hkv * D], -1))
    if s['cos'] is not None:
        # keys in 64 bits: a rounding of theirs may land next to a border between two codes
        q, k = (_rotated(q, s['cos'], s['sin'], s['interleaved']).to(q.dtype),
                _rotated(k, s['cos'].double(), s['sin'].double(), s['interleaved']))
    slots, nb = s['slots'], D // 32
    tiles = s['k_cache'].shape[2]
    BS = 16 * tiles
    # byte offset of each token's tile, per head
    tile = (((slots // BS)[:, None] * Hkv + torch.arange(Hkv, device=slots.device)) * tiles
            + (slots % BS // 16)[:, None]) * (17 * D // 2)
    tile, r = tile[..., None], (slots % 16)[:, None, None]
    c, b = torch.arange(D // 2, device=slots.device), torch.arange(nb, device=slots.device)
    kc, ks = _quantise(k)
    vc, vs = _quantise(v.float())
    flat_k, flat_v = s['k_cache'].view(-1), s['v_cache'].view(-1)
    flat_k[tile + r * (D // 2) + c] = kc[..., 0::2] | kc[..., 1::2] << 4
    flat_k[tile + 8 * D + r * nb + b] = ks
    flat_v[tile + ((r // 4 * 16 + c % 16) * nb + c // 16) * 4 + r % 4] = vc[..., 0::2] | vc[..., 1::2] << 4
    flat_v[tile + 8 * D + (r // 4 * nb + b) * 4 + r % 4] = vs
    return dict(q=q.contiguous(), k=_values(kc, ks).to(q.dtype), v=_values(vc, vs).to(q.dtype))


def _gathered(cache, tables, value_form):
    """A cache's rows by block table: float32 [sequences, heads, tokens, D]."""
    rows = _values(*_unpack(cache[tables.long()], value_form))       # [n, blocks, H, tiles, 16, D]
    return rows.permute(0, 2, 1, 3, 4, 5).flatten(2, 4)


def _plain_decode(s):
    q = s['q'].float()
    B, Hq, D = q.shape
    k, v = _gathered(s['k_cache'], s['tables'], False), _gathered(s['v_cache'], s['tables'], True)
    live = (torch.arange(k.shape[2], device=q.device) < s['lens'][:, None])[:, None, None]
    score = q.view(B, k.shape[1], -1, D) @ k.transpose(-1, -2) * D ** -0.5
    score = torch.where(live, score, torch.full_like(score, -math.inf))
    p = torch.exp(score - score.amax(-1, keepdim=True))
    v = torch.where(live.transpose(-1, -2), v, torch.zeros_like(v))
    return ((p @ v) / p.sum(-1, keepdim=True)).view(B, Hq, D).to(s['q'].dtype)


def _plain_chunk(s):
    D, Hkv = s['q'].shape[2], s['k_cache'].shape[1]
    start, _, pos0 = s['meta'].long()
    k, v = _gathered(s['k_cache'], s['tables'], False), _gathered(s['v_cache'], s['tables'], True)
    at = torch.arange(s['longest'], device=k.device)
    rows = s['q'].float()[(start[:, None] + at).clamp(max=s['q'].shape[0] - 1)]     # [n, longest, Hq, D]
    rows = rows.unflatten(2, (Hkv, -1)).permute(0, 2, 3, 1, 4)                       # [n, Hkv, G, longest, D]
    score = (rows.flatten(2, 3) @ k.transpose(-1, -2)).view(*rows.shape[:4], -1) * D ** -0.5
    live = torch.arange(k.shape[2], device=k.device) <= (pos0[:, None] + at)[:, :, None]
    score = torch.where(live[:, None, None], score, torch.full_like(score, -math.inf))
    p = torch.exp(score - score.amax(-1, keepdim=True))
    v = torch.where(live.any(1)[:, None, :, None], v, torch.zeros_like(v))
    out = (p.flatten(2, 3) @ v).view(rows.shape) / p.sum(-1, keepdim=True)
    return out.permute(0, 3, 1, 2, 4).flatten(2, 3)[s['seg'], s['off']].to(s['q'].dtype)


# ---------------------------------------------------------------------------------------------- one pass
def run(s):
    if own:
        ops = _ops()
        if s['op'] == 'angles':
            cos, sin = ops.rope_angles(s['positions'], s['freq'], s['factor'])
            return dict(cos=cos, sin=sin)
        if s['op'] == 'append':
            T, Hq, Hkv, D = s['qkv'].shape[0], s['Hq'], s['Hkv'], s['D']
            q, k, v = (t.view(T, -1, D) for t in s['qkv'].split([Hq * D, Hkv * D, Hkv * D], -1))
            q = ops.rope_kv4_write(q, k, v, s['cos'], s['sin'], s['slots'], s['k_cache'], s['v_cache'],
                                   interleaved=s['interleaved'])
            k, v = ops.kv4_read_slots(s['k_cache'], s['v_cache'], s['slots'], q.dtype)
            return dict(q=q, k=k, v=v)
        if s['op'] == 'decode':
            return ops.paged_decode_kv4(s['q'], s['k_cache'], s['v_cache'], s['tables'], s['lens'], s['longest'])
        return ops.paged_prefill_kv4(s['q'], s['k_cache'], s['v_cache'], s['tables'], s['meta'][0], s['meta'][1],
                                     s['meta'][2], s['longest'], s['context'])
    return dict(angles=_plain_angles, append=_plain_append, decode=_plain_decode, chunk=_plain_chunk)[s['op']](s)


# ---------------------------------------------------------------------------------------------- from the definition, 64 bits
def _nearest(x):
    """x [..., 32 n] rounded to the cache's values: per 32 dims a power of two with the largest at most 6 times it, then
    the nearest of the E2M1 values, ties to the one with an even code."""
    x = x.double().unflatten(-1, (-1, 32))
    top = x.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(top / 6)).clamp(-120, 125)
    e = e + (top > 6 * 2.0 ** e).double() - (top <= 3 * 2.0 ** e).double()
    e = torch.where(top > 0, e.clamp(-120, 125), torch.zeros_like(e))
    a = x.abs() / 2.0 ** e
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0)).double()
    return (x.sign() * (torch.round(a / step) * step).clamp(max=6) * 2.0 ** e).flatten(-2)


def _row(cache, block, t, value_form):
    """Tokens t [n] of a sequence with block ids `block` -> float64 [heads, n, D], from the bytes' places."""
    BS, D = 16 * cache.shape[2], cache.shape[3] * 2 // 17
    nb, d = D // 32, torch.arange(D, device=cache.device)
    record = cache[block[t // BS].long(), :, t % BS // 16]                       # [n, heads, bytes]
    r = (t % 16)[:, None]
    if value_form:
        at = ((r // 4 * 16 + d % 32 // 2) * nb + d // 32) * 4 + r % 4
        scale_at = 8 * D + (r // 4 * nb + d // 32) * 4 + r % 4
    else:
        at, scale_at = r * (D // 2) + d // 2, 8 * D + r * nb + d // 32
    H = record.shape[1]
    byte = record.gather(2, at[:, None].expand(-1, H, -1)).long()
    scale = record.gather(2, scale_at[:, None].expand(-1, H, -1)).double()
    code = byte // torch.where(d % 2 == 1, 16, 1) % 16
    m, e = code % 2, code // 2 % 4
    size = torch.where(e == 0, m * 0.5, (1 + m * 0.5) * 2.0 ** (e - 1.0))
    return (torch.where(code >= 8, -size, size) * 2.0 ** (scale - 127)).transpose(0, 1)


def _attend(q, k, v, live, D):
    """q [Hkv, rows, D], k / v [Hkv, n, D], live [rows, n] or None."""
    score = torch.matmul(q, k.transpose(1, 2)) / math.sqrt(D)
    if live is not None:
        score = score.masked_fill(~live, -math.inf)
    return torch.matmul(torch.softmax(score, -1), v)


def exact(case, seed):
    s = prepare(case, seed)
    if case['op'] == 'angles':
        ang = s['positions'].double()[:, None] * s['freq']
        return dict(cos=torch.cos(ang) * s['factor'], sin=torch.sin(ang) * s['factor'])
    D = case['D']
    if case['op'] == 'append':
        T, Hq, Hkv = case['T'], case['Hq'], case['Hkv']
        x = s['qkv'].double().view(T, Hq + 2 * Hkv, D)
        turned = x[:, :Hq + Hkv].clone()
        half = case['rotary'] // 2
        for i in range(half):
            a, b = (2 * i, 2 * i + 1) if case['interleaved'] else (i, i + half)
            c, w = s['cos'][:, i, None].double(), s['sin'][:, i, None].double()
            turned[..., a] = x[:, :Hq + Hkv, a] * c - x[:, :Hq + Hkv, b] * w
            turned[..., b] = x[:, :Hq + Hkv, b] * c + x[:, :Hq + Hkv, a] * w
        return dict(q=turned[:, :Hq], k=_nearest(turned[:, Hq:]), v=_nearest(x[:, Hq + Hkv:]))
    Hq, Hkv = case['Hq'], case['Hkv']
    if case['op'] == 'decode':
        lens, pos0 = [1] * case['B'], [n - 1 for n in _lengths(case)]
    else:
        lens, pos0 = _lengths(case)
    out, at = [], 0
    for i, (n, p) in enumerate(zip(lens, pos0)):
        t = torch.arange(n + p, device='cuda')
        k, v = _row(s['k_cache'], s['tables'][i], t, False), _row(s['v_cache'], s['tables'][i], t, True)
        q = s['q'][at:at + n].double().view(n, Hkv, -1, D).transpose(0, 1).flatten(1, 2)        # rows (token, head of the group)
        live = (t <= p + torch.arange(n, device='cuda')[:, None]).repeat_interleave(Hq // Hkv, 0)
        out.append(_attend(q, k, v, live, D).view(Hkv, n, -1, D).transpose(0, 1).reshape(n, Hq, D))
        at += n
    return torch.cat(out)
