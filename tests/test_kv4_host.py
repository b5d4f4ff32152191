"""The 4-bit KV cache without a GPU: the checker's format against hand-worked values, the host-side
arithmetic of rope_frequencies, and every refusal of the C entry points (argument checks come before
any device work)."""
import math

import numpy as np
import pytest
import torch

from mi355_paged import _lib, ops
from oracle import kv4_oracle as orc


# ------------------------------------------------------------------ format
def test_codes_round_to_nearest_with_ties_to_the_even_code():
    a = [0.0, 0.25, 0.2500001, 0.75, 0.7499999, 1.25, 1.2500001, 1.75, 2.5, 2.5000001, 3.5, 3.4999999, 5.0, 5.0000001, 9.0]
    want = [0, 0, 1, 2, 1, 2, 3, 4, 4, 5, 6, 5, 6, 7, 7]
    assert orc.round_code(a).tolist() == want


def test_scales_are_the_smallest_power_of_two_that_holds_the_block():
    x = np.zeros((6, 32))
    x[0, 3], x[1, 5], x[2, 0], x[3, 31] = 6.0, 6.0000001, -3.0, 3.0000001
    x[4, 1] = np.nan
    code, byte = orc.quantise(x)
    assert byte[:, 0].tolist() == [127, 128, 126, 127, 255, 127 + orc.MIN_EXP]
    v = orc.dequantise(code, byte)
    assert v[0, 3] == 6.0 and v[1, 5] == 6.0 and v[2, 0] == -3.0 and v[3, 31] == 3.0
    assert np.isnan(v[4]).all() and not v[5].any()


@pytest.mark.parametrize('D', [32, 64, 128, 256])
@pytest.mark.parametrize('value_form', [False, True])
def test_every_code_and_scale_has_a_place_of_its_own(D, value_form):
    places = {(a, s) for r in range(16) for d in range(D) for a, s in [orc.code_place(D, r, d, value_form)]}
    assert len(places) == 16 * D and max(a for a, _ in places) == 8 * D - 1
    scales = {orc.scale_place(D, r, b, value_form) for r in range(16) for b in range(D // 32)}
    assert scales == set(range(8 * D, 17 * D // 2))
    rng = np.random.default_rng(D)
    code = rng.integers(0, 16, (3, 16, D)).astype(np.uint8)
    byte = rng.integers(100, 140, (3, 16, D // 32)).astype(np.uint8)
    rec = orc.pack(code, byte, value_form)
    assert rec.shape[-1] == ops.kv4_cache_shape(1, 1, 16, D)[3] == orc.record_bytes(D)
    np.testing.assert_array_equal(orc.unpack(rec, value_form), orc.dequantise(code, byte))
    one = np.zeros(orc.record_bytes(D), dtype=np.uint8)
    for r in range(16):
        orc.write_row(one, r, code[0, r], byte[0, r], value_form)
    np.testing.assert_array_equal(one, rec[0])


def test_cache_shape_refuses_what_the_format_does_not_hold():
    assert ops.kv4_cache_shape(7, 3, 48, 64) == (7, 3, 3, 544)
    with pytest.raises(ValueError, match='head_dim'):
        ops.kv4_cache_shape(7, 3, 16, 48)
    for bs in (0, 8, 24, -16):
        with pytest.raises(ValueError, match='tiles of 16'):
            ops.kv4_cache_shape(7, 3, bs, 64)


# ------------------------------------------------------------------ frequencies
def test_rope_frequencies():
    f, factor = ops.rope_frequencies(8)
    assert f.dtype == torch.float64 and factor == 1.0
    np.testing.assert_allclose(f.numpy(), [1.0, 0.1, 0.01, 0.001], rtol=1e-15)
    lin, factor = ops.rope_frequencies(8, scaling={'kind': 'linear', 'factor': 4})
    np.testing.assert_allclose(lin.numpy(), f.numpy() / 4, rtol=1e-15)
    assert factor == 1.0
    ntk, _ = ops.rope_frequencies(8, scaling={'kind': 'ntk', 'factor': 4})
    assert ntk[0] == 1.0
    np.testing.assert_allclose(float(ntk[-1]), float(f[-1]) / 4, rtol=1e-12)
    yarn, factor = ops.rope_frequencies(64, scaling={'kind': 'yarn', 'factor': 8, 'original': 4096})
    plain, _ = ops.rope_frequencies(64)
    turns = plain.numpy() * 4096 / (2 * math.pi)
    assert factor == 0.1 * math.log(8) + 1
    for i in range(32):
        keep = min(1.0, max(0.0, (turns[i] - 1) / 31))
        np.testing.assert_allclose(float(yarn[i]), plain[i] * keep + plain[i] / 8 * (1 - keep), rtol=1e-14)
    assert (turns > 32).any() and (turns < 1).any()


@pytest.mark.parametrize('args', [dict(rotary_dim=7), dict(rotary_dim=0), dict(rotary_dim=8, scaling={'kind': 'other'}),
                                  dict(rotary_dim=8, scaling={'kind': 'linear', 'factor': 0}),
                                  dict(rotary_dim=2, scaling={'kind': 'ntk', 'factor': 2}),
                                  dict(rotary_dim=8, scaling={'kind': 'yarn', 'factor': 2}),
                                  dict(rotary_dim=8, scaling={'kind': 'yarn', 'factor': 2, 'original': 10, 'beta_slow': 40})])
def test_rope_frequencies_refuses(args):
    with pytest.raises(ValueError):
        ops.rope_frequencies(**args)


# ------------------------------------------------------------------ refusals (no device is touched)
P = 4096            # a well aligned address that no refused call reads
OUT = 1 << 24       # one behind it
LONG = (1 << 31) - 1


def _call(name, good, **change):
    args = dict(good, **change)
    rc = getattr(_lib.load(), name)(*args.values())
    return rc, _lib.load().mi355_last_error().decode()


ANGLES = dict(cos=P, sin=P, positions=P, freq=P, factor=1.0, T=4, half=8, stream=None)
ROTATE = dict(out=OUT, x=P, stride=8 * 64, cos=P, sin=P, R=64, inter=0, T=4, H=8, D=64, dtype=1, stream=None)
WRITE = dict(q_out=OUT, q=P, k=P, v=P, qs=1536, ks=1536, vs=1536, cos=P, sin=P, R=64, inter=0, slots=P, kc=P, vc=P, T=4,
             Hq=8, Hkv=8, D=64, BS=16, NB=10, sb=8 * 544, sh=544, dtype=1, stream=None)
READ = dict(ko=P, vo=P, kc=P, vc=P, slots=P, T=4, Hkv=8, D=64, BS=16, NB=10, sb=8 * 544, sh=544, dtype=1, stream=None)
DECODE = dict(out=P, q=P, qs=512, kc=P, vc=P, bt=P, ctx=P, B=2, Hq=8, Hkv=8, D=64, BS=16, mb=4, NB=10, max_ctx=64,
              sb=8 * 544, sh=544, scale=0.125, dtype=1, ws=P, wsb=1 << 30, stream=None)
CHUNK = dict(out=P, q=P, qs=512, kc=P, vc=P, bt=P, q0=P, ln=P, pos=P, nseg=2, rows=16, max_q=8, Hq=8, Hkv=8, D=64, BS=16, mb=4,
             NB=10, max_ctx=64, sb=8 * 544, sh=544, scale=0.125, dtype=1, ws=P, wsb=1 << 30, stream=None)
CACHE = [(dict(kc=None), -1), (dict(vc=None), -1), (dict(kc=P + 8), -1), (dict(D=16), -2), (dict(D=96), -2), (dict(BS=8), -2),
         (dict(BS=24), -2), (dict(BS=0), -2), (dict(NB=0), -1), (dict(Hkv=0), -1), (dict(sh=540), -1), (dict(sb=8), -1),
         (dict(sh=528), -1), (dict(sb=528), -1), (dict(dtype=3), -1), (dict(sh=-544), -1)]
REFUSED = (
    [('mi355_rope_angles', ANGLES, c, -1) for c in (dict(cos=None), dict(sin=None), dict(positions=None), dict(freq=None),
                                                  dict(T=-1), dict(half=0), dict(T=LONG))] +
    [('mi355_rope_rotate', ROTATE, c, r) for c, r in (
        (dict(out=None), -1), (dict(x=None), -1), (dict(cos=None), -1), (dict(sin=None), -1), (dict(R=8), -1), (dict(R=80), -1),
        (dict(R=-16), -1), (dict(T=-1), -1), (dict(H=0), -1), (dict(D=48), -2), (dict(dtype=7), -1), (dict(stride=504), -1),
        (dict(stride=516), -1), (dict(x=P + 4), -1), (dict(out=OUT + 2), -1), (dict(cos=P + 4), -1), (dict(T=LONG), -1),
        (dict(out=P), -1), (dict(out=P + 4 * 1024 - 16), -1), (dict(x=OUT + 4 * 1024 - 16), -1))] +
    [('mi355_rope_kv4_write', WRITE, c, r) for c, r in CACHE + [
        (dict(q_out=None), -1), (dict(q=None), -1), (dict(k=None), -1), (dict(v=None), -1), (dict(slots=None), -1),
        (dict(ks=504), -1), (dict(vs=1540), -1), (dict(k=P + 2), -1), (dict(Hq=0), -1), (dict(R=24), -1), (dict(cos=None), -1),
        (dict(T=-3), -1), (dict(T=LONG), -1), (dict(q_out=P), -1), (dict(k=OUT + 2048), -1), (dict(v=OUT - 3 * 2 * 1536 - 512), -1)]] +
    [('mi355_kv4_read_slots', READ, c, r) for c, r in CACHE + [
        (dict(ko=None), -1), (dict(vo=P + 8), -1), (dict(slots=None), -1), (dict(T=-1), -1), (dict(T=LONG), -1)]] +
    [('mi355_paged_decode_kv4', DECODE, c, r) for c, r in CACHE + [
        (dict(out=None), -1), (dict(q=None), -1), (dict(bt=None), -1), (dict(ctx=None), -1), (dict(qs=504), -1), (dict(qs=516), -1),
        (dict(q=P + 8), -1), (dict(Hq=12), -1), (dict(Hq=0), -1), (dict(B=-1), -1), (dict(mb=0), -1), (dict(max_ctx=-1), -1),
        (dict(max_ctx=100000, mb=7000, ws=None), -3), (dict(max_ctx=100000, mb=7000, wsb=64), -3),
        (dict(max_ctx=100000, mb=7000, ws=P + 4), -3), (dict(max_ctx=1 << 30, mb=1 << 27), -1), (dict(B=1 << 24), -1)]] +
    [('mi355_paged_prefill_kv4', CHUNK, c, r) for c, r in CACHE + [
        (dict(out=None), -1), (dict(q=None), -1), (dict(bt=None), -1), (dict(q0=None), -1), (dict(ln=None), -1), (dict(pos=None), -1),
        (dict(qs=504), -1), (dict(q=P + 8), -1), (dict(Hq=12), -1), (dict(nseg=-1), -1), (dict(max_q=-1), -1), (dict(mb=0), -1),
        (dict(max_ctx=0), -1), (dict(max_q=1 << 30, rows=1 << 30, Hq=64, qs=4096), -1), (dict(nseg=1 << 20, rows=1 << 20, max_q=1 << 16), -1), (dict(rows=-1), -1),
        (dict(max_ctx=100000, mb=7000, ws=None), -3), (dict(max_ctx=100000, mb=7000, wsb=64), -3),
        (dict(max_ctx=100000, mb=7000, ws=P + 4), -3), (dict(max_ctx=1 << 30, mb=1 << 27), -1)]])


@pytest.mark.parametrize('name,good,change,want', REFUSED, ids=lambda v: str(v)[:40])
def test_c_entry_points_refuse(name, good, change, want):
    rc, message = _call(name, good, **change)
    assert rc == want, (rc, message)
    assert name.replace('mi355_', '') in message


@pytest.mark.parametrize('name,good', [('mi355_paged_decode_kv4', DECODE), ('mi355_paged_prefill_kv4', CHUNK)])
@pytest.mark.parametrize('out,qs,dtype', [(P + 1024, 512, 1), (P - 1024, 512, 2), (P, 1536, 1), (P + 512 * 4, 1536, 0), (P + 2048 - 16, 512, 1)])
def test_outputs_that_overlap_the_queries_are_refused(name, good, out, qs, dtype):
    rows = dict(B=2) if 'B' in good else dict(rows=2)
    rc, message = _call(name, good, out=out, qs=qs, dtype=dtype, **rows)
    assert rc == -1 and 'overlaps' in message


@pytest.mark.parametrize('name,good,empty', [
    ('mi355_rope_angles', ANGLES, dict(T=0, cos=None)), ('mi355_rope_rotate', ROTATE, dict(T=0, x=None)),
    ('mi355_rope_kv4_write', WRITE, dict(T=0, q=None, slots=None)), ('mi355_kv4_read_slots', READ, dict(T=0, ko=None)),
    ('mi355_paged_decode_kv4', DECODE, dict(B=0, q=None)), ('mi355_paged_prefill_kv4', CHUNK, dict(nseg=0, q=None)),
    ('mi355_paged_prefill_kv4', CHUNK, dict(max_q=0))])
def test_empty_calls_do_nothing(name, good, empty):
    assert _call(name, good, **empty)[0] == 0


def test_workspace_queries_are_host_arithmetic():
    lib = _lib.load()
    assert lib.mi355_paged_decode_kv4_workspace_bytes(1, 8, 8, 64, 37, 1) == 0            # one split
    assert lib.mi355_paged_decode_kv4_workspace_bytes(1, 8, 8, 64, 100000, 1) > 0
    assert lib.mi355_paged_decode_kv4_workspace_bytes(1, 8, 8, 48, 100000, 1) == 0        # refused: the call says why
    assert lib.mi355_paged_prefill_kv4_workspace_bytes(1, 8, 8, 8, 8, 64, 100000, 1) > 0
    assert lib.mi355_paged_prefill_kv4_workspace_bytes(8, 8192, 1024, 8, 8, 64, 1024, 1) == 0
    assert lib.mi355_paged_prefill_kv4_workspace_bytes(1, 8, 1 << 30, 8, 8, 64, 100000, 1) == \
        lib.mi355_paged_prefill_kv4_workspace_bytes(1, 8, 8, 8, 8, 64, 100000, 1)              # no more rows than there are


def test_ops_refuse_host_tensors():
    k = torch.zeros(ops.kv4_cache_shape(2, 2, 16, 32), dtype=torch.uint8)
    with pytest.raises(RuntimeError, match='HIP device'):
        ops.kv4_read_slots(k, k, torch.zeros(1, dtype=torch.int64))
    with pytest.raises(RuntimeError, match='HIP device'):
        ops.rope_angles(torch.zeros(1, dtype=torch.int64), torch.zeros(4, dtype=torch.float64))


def test_blocks_beyond_the_entry_points_integers_are_refused():
    big = torch.empty((1, 1, (1 << 28) + 1, 17 * 32 // 2), dtype=torch.uint8, device='meta')     # (16 tokens to a 32-bit count)
    with pytest.raises(ValueError, match='per block'):
        ops._kv4_geometry(big, big)
    assert ops._kv4_geometry(big[:, :, :1000], big[:, :, :1000])[2] == 16000


# ------------------------------------------------------------------ the engine's arguments
@pytest.mark.parametrize('kw', [dict(kv_cache_dtype='mxfp4'), dict(rotary={}), dict(kv_cache_dtype='mxfp4', device='cuda', reference_compat=True),
                                dict(kv_cache_dtype='fp4', device='cuda')])
def test_engine_refuses_settings_it_does_not_serve(kw):
    import mini_vllm
    with pytest.raises(ValueError):
        mini_vllm.MiniVLLM(**kw)


@pytest.mark.parametrize('kw,match', [(dict(num_heads=8), 'head_dim'), (dict(block_size=8), 'tiles of 16'), (dict(rotary=dict(dim=24)), 'multiple of 16'),
                                      (dict(rotary=dict(dim=64)), 'head_dim'), (dict(rotary=dict(scaling={'kind': 'x'})), 'scaling kind'),
                                      (dict(kv_cache_dtype='int4'), 'mxfp4')])
def test_model_refuses_what_the_cache_does_not_hold(kw, match):
    import mini_vllm
    args = dict(vocab_size=50, hidden_size=128, num_layers=1, num_heads=4, intermediate_size=64, num_kv_blocks=4, block_size=16,
                kv_cache_dtype='mxfp4')
    with pytest.raises(ValueError, match=match):
        mini_vllm.MiniTransformer(**dict(args, **kw))


def test_model_holds_the_caches_it_announces():
    import mini_vllm
    m = mini_vllm.MiniTransformer(50, 128, 2, 4, 64, 6, 32, kv_cache_dtype='mxfp4')
    assert m.k_cache.shape == m.v_cache.shape == (2, 6, 4, 2, 17 * 32 // 2) and m.k_cache.dtype == torch.uint8
    assert m.to(torch.bfloat16).k_cache.dtype == torch.uint8
    plain = mini_vllm.MiniTransformer(50, 128, 2, 4, 64, 6, 32)
    assert plain.k_cache.shape == (2, 6, 32, 4, 32) and plain.k_cache.dtype == torch.float32


def test_plan_keeps_prompts_on_the_cache():
    import mini_vllm
    args = dict(positions=list(range(5)) + [7] + [0], seq_lens=[5, 1, 1], is_prefill=[True, False, True],
                block_tables=[[0], [1], [2]], device='cpu', append_ok=True)
    plan = mini_vllm.build_attn_plan(**args, from_cache=True)
    assert plan.causal_tokens == 0 and plan.append_tokens == 5 and plan.append_meta.tolist() == [[0], [5], [0]]
    assert plan.paged_rows == 2 and plan.paged_context.tolist() == [8, 1] and not plan.pure_decode
    assert mini_vllm.build_attn_plan(**args).causal_tokens == 6


@pytest.mark.parametrize('kw', [dict(), dict(reference_compat=True, block_tables=[[0]]), dict(table_rows=[0])])
@pytest.mark.parametrize('prefill', [True, False])
def test_model_over_a_4_bit_cache_needs_block_tables(kw, prefill):
    """Without them a decode token would attend to slot 0 alone (the reference's decode branch), without an error."""
    import mini_vllm
    model = mini_vllm.MiniTransformer(50, 128, 1, 4, 64, 4, 16, kv_cache_dtype='mxfp4')
    one = torch.zeros(1, dtype=torch.int64)
    with pytest.raises(ValueError, match='block tables'):
        model(one, one, one, [1], [prefill], **kw)


def test_layer_over_a_4_bit_cache_needs_a_plan():
    import mini_vllm
    model = mini_vllm.MiniTransformer(50, 128, 1, 4, 64, 4, 16, kv_cache_dtype='mxfp4')
    one = torch.zeros(1, dtype=torch.int64)
    with pytest.raises(ValueError, match='block tables'):
        model.layers[0].attn(torch.zeros(1, 128), one, (model.k_cache[0], model.v_cache[0]), one, [1], [False])
