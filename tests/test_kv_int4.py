"""The 4-bit KV cache without a GPU: the format against hand-made rows, what the entry points refuse, and where a row stands."""
import subprocess

import numpy as np
import pytest

from conftest import ROOT

PTR = 4096          # a made-up aligned address: every call below is refused before anything is launched


def test_pack_places_and_round_trip(oracle):
    for d in range(32, 257, 32):
        word, shift = oracle.kv4_places(d)
        assert len(set(zip(word, shift))) == d and word.max() == d // 8 - 1
        codes = np.random.default_rng(d).integers(0, 16, (3, d))
        assert (oracle.kv4_unpack(oracle.kv4_pack(codes)) == codes).all()
    codes = np.zeros((1, 128), dtype=np.int64)
    codes[0, 4 * 9] = 5                # unit 9 = 8 * 1 + 1: place 1 * 4 + 1 = 5, the upper half of word 2
    assert oracle.kv4_pack(codes)[0].tolist() == [0, 0, 5 << 16] + [0] * 13


def test_quantise_known_rows(oracle):
    ramp = np.arange(32, dtype=np.float16)[None] / 2                    # 0 .. 15.5, scale 15.5 / 15
    w, p = oracle.kv4_quantise(ramp, 32)
    assert p[0, 0].tolist() == [float(np.float16(15.5 / 15)), 0.0]
    flat = np.full((1, 32), -3.5, dtype=np.float16)
    w, p = oracle.kv4_quantise(flat, 32)
    assert (oracle.kv4_unpack(w) == 0).all() and (oracle.kv4_values(w, p) == -3.5).all()
    ties = np.concatenate([[0, 15], np.arange(15) + 0.5, np.zeros(15)]).astype(np.float16)[None]   # scale 1: every border
    w, p = oracle.kv4_quantise(ties, 32)
    assert oracle.kv4_unpack(w)[0, 2:17].tolist() == [2 * ((i + 1) // 2) for i in range(15)]        # to the even code
    big = np.array([[np.inf, -np.inf] + [0.0] * 30])
    w, p = oracle.kv4_quantise(big, 32)
    v = oracle.kv4_values(w, p)
    assert np.isfinite(v).all() and np.isfinite(v.astype(np.float16)).all() and v[0, 1] == -65440
    nan = np.zeros((1, 64), dtype=np.float32)
    nan[0, 3] = np.nan
    v = oracle.kv4_values(*oracle.kv4_quantise(nan, 32))
    assert np.isnan(v[0, :32]).all() and (v[0, 32:] == 0).all()


def _append(L, **kw):
    a = dict(nk=PTR, nv=PTR, kc=PTR, kp=PTR, vc=PTR, vp=PTR, idx=PTR, new=None, heads=8, d=128, g=64, ml=100, b=2, t=3, sk=1024, sv=1024)
    a.update(kw)
    L.call("kv_cache_append_hm_int4_f16", *a.values(), None)


def _append_paged(L, **kw):
    a = dict(nk=PTR, nv=PTR, kc=PTR, kp=PTR, vc=PTR, vp=PTR, table=PTR, idx=PTR, new=None, heads=8, d=128, g=64, bs=16, nb=9, mb=4, b=2, t=3,
             sk=1024, sv=1024)
    a.update(kw)
    L.call("kv_cache_append_paged_int4_bf16", *a.values(), None)


def _rope(L, **kw):
    a = dict(qkv=PTR, cos=PTR, sin=PTR, pos=PTR, qo=PTR, kc=PTR, kp=PTR, vc=PTR, vp=PTR, hq=32, heads=8, d=128, g=64, ml=100, b=2)
    a.update(kw)
    L.call("rope_kv_append_hm_int4_bf16", *a.values(), None)


def _read(L, **kw):
    a = dict(kc=PTR, kp=PTR, vc=PTR, vp=PTR, first=None, lens=PTR, ko=PTR, vo=PTR, heads=8, d=128, g=64, ml=100, b=2, ol=10)
    a.update(kw)
    L.call("kv_cache_read_hm_int4_f16", *a.values(), None)


def _attn(L, **kw):
    a = dict(q=PTR, kc=PTR, kp=PTR, vc=PTR, vp=PTR, lens=PTR, out=PTR, b=2, hq=32, heads=8, d=128, g=64, ml=100, scale=0.1, ws=PTR, wb=1 << 30)
    a.update(kw)
    L.call("batched_decode_attention_hm_int4_f16_ws", *a.values(), None)


def _attn_paged(L, **kw):
    a = dict(q=PTR, kc=PTR, kp=PTR, vc=PTR, vp=PTR, table=PTR, lens=PTR, out=PTR, b=2, hq=32, heads=8, d=128, g=64, bs=16, nb=9, mb=4, scale=0.1,
             ws=PTR, wb=1 << 30)
    a.update(kw)
    L.call("batched_decode_attention_paged_int4_bf16_ws", *a.values(), None)


NULL, SHAPE, ALIGN, WORKSPACE = -1, -2, -3, -4


@pytest.mark.parametrize("call,kw,code", [
    *[(f, kw, code) for f in (_append, _append_paged, _rope, _read, _attn, _attn_paged) for kw, code in [
        (dict(kc=None), NULL), (dict(kp=None), NULL), (dict(vc=None), NULL), (dict(vp=None), NULL), (dict(heads=0), SHAPE), (dict(d=0), SHAPE),
        (dict(d=48), SHAPE), (dict(d=288), SHAPE), (dict(d=96), SHAPE), (dict(g=16), SHAPE), (dict(g=0), SHAPE), (dict(g=256, d=256), SHAPE),
        (dict(b=-1), SHAPE), (dict(b=65536), SHAPE), (dict(kc=PTR + 4), ALIGN), (dict(vp=PTR + 8), ALIGN)]],
    *[(f, kw, SHAPE) for f in (_append, _rope, _read, _attn) for kw in (dict(ml=0), dict(ml=-5), dict(ml=2 ** 30 + 1))],
    *[(f, kw, code) for f in (_append_paged, _attn_paged) for kw, code in [
        (dict(table=None), NULL), (dict(bs=0), SHAPE), (dict(nb=0), SHAPE), (dict(mb=0), SHAPE), (dict(bs=1 << 16, mb=1 << 15), SHAPE)]],
    *[(f, kw, code) for f in (_append, _append_paged) for kw, code in [
        (dict(nk=None), NULL), (dict(nv=None), NULL), (dict(idx=None), NULL), (dict(t=-1), SHAPE), (dict(sk=1016), SHAPE), (dict(sv=0), SHAPE),
        (dict(sk=1028), ALIGN), (dict(nk=PTR + 8), ALIGN)]],
    *[(_rope, kw, code) for kw, code in [(dict(qkv=None), NULL), (dict(cos=None), NULL), (dict(sin=None), NULL), (dict(pos=None), NULL),
                                         (dict(qo=None), NULL), (dict(hq=0), SHAPE), (dict(qkv=PTR + 2), ALIGN), (dict(qo=PTR + 8), ALIGN)]],
    *[(_read, kw, code) for kw, code in [(dict(lens=None), NULL), (dict(ko=None), NULL), (dict(vo=None), NULL), (dict(ol=-1), SHAPE),
                                         (dict(ko=PTR + 8), ALIGN)]],
    *[(f, kw, code) for f in (_attn, _attn_paged) for kw, code in [
        (dict(q=None), NULL), (dict(lens=None), NULL), (dict(out=None), NULL), (dict(hq=0), SHAPE), (dict(hq=30), SHAPE), (dict(q=PTR + 2), ALIGN),
        (dict(out=PTR + 8), ALIGN), (dict(wb=1024), WORKSPACE), (dict(ws=PTR + 8), WORKSPACE)]],
])
def test_refusals(pkg, call, kw, code):
    with pytest.raises(pkg.B200KError) as e:
        call(pkg.lib(), **kw)
    assert e.value.code == code, e.value.message


def test_head_counts_whose_sum_passes_32_bits(pkg):
    for hq, heads in ((2 ** 31 - 1, 2 ** 30), (2 ** 31 - 1, 2 ** 30 + 8), (2 ** 30, 8), (32, 2 ** 31 - 1)):
        with pytest.raises(pkg.B200KError) as e:
            _rope(pkg.lib(), hq=hq, heads=heads)
        assert e.value.code == SHAPE


def test_layer_cache_refusals(pkg):
    L = pkg.lib()
    for args, code in ([(None, PTR, PTR, PTR, PTR, 64), NULL], [(PTR, None, PTR, PTR, PTR, 64), NULL], [(PTR, PTR, PTR, PTR, None, 64), NULL],
                       [(PTR, PTR, PTR, PTR, PTR, 48), SHAPE], [(PTR, PTR, PTR + 4, PTR, PTR, 64), ALIGN]):
        with pytest.raises(pkg.B200KError) as e:
            L.call("b200k_layer_set_kv_cache_int4", *args)
        assert e.value.code == code


def test_cache_tensors(pkg):
    codes, params = pkg.prelude.int4_kv_cache(3, 2, 5, 96, 32, "cpu")
    assert codes.shape == (3, 2, 5, 12) and params.shape == (3, 2, 5, 3, 2)
    for d, g in ((100, 32), (96, 64)):
        with pytest.raises(ValueError):
            pkg.prelude.int4_kv_cache(1, 1, 1, d, g, "cpu")


def test_empty_calls_launch_nothing(pkg):
    L = pkg.lib()
    _append(L, b=0); _append(L, t=0); _append_paged(L, b=0); _rope(L, b=0); _read(L, b=0); _read(L, ol=0); _attn(L, b=0); _attn_paged(L, b=0)
    assert L.call("b200k_attention_int4_workspace_bytes", 0, 32, 8, 128) == 0
    assert L.call("b200k_attention_int4_workspace_bytes", 4, 32, 8, 128) >= 128 * 1024


def test_row_addresses_and_bad_blocks(tmp_path):
    """The function that places a row, compiled for the host: every table entry outside the pool gives -1, and a far row of a
    long cache has a 64-bit index."""
    src = tmp_path / "rows.cu"
    src.write_text('''
#include "%s/triton-rs_b200/csrc/kv_int4.cuh"
using namespace b200k;
int main() {
    Kv4Cache C = kv4_cache(nullptr, nullptr, nullptr, nullptr, 8, 128, 64, 1 << 20);
    if (kv4_row(C, 0, 0, 0) != 0 || kv4_row(C, 1, 2, 3) != ((1l * 8 + 2) << 20) + 3) return 1;
    if (kv4_row(C, 4000, 7, (1 << 20) - 1) != ((4000l * 8 + 8) << 20) - 1) return 2;
    const int table[2][3] = {{5, 0, 2}, {-1, 6, 1 << 30}};
    Kv4Cache P = kv4_pool(nullptr, nullptr, nullptr, nullptr, &table[0][0], 4, 128, 64, 16, 6, 3);
    if (P.capacity != 48) return 3;
    if (kv4_row(P, 0, 3, 15) != (5 * 4 + 3) * 16 + 15 || kv4_row(P, 0, 1, 16) != (0 * 4 + 1) * 16 || kv4_row(P, 0, 0, 47) != 2 * 4 * 16 + 15) return 4;
    for (int pos = 0; pos < 48; ++pos)
        if (kv4_row(P, 1, 2, pos) != -1) return 5;      // below 0, one past the pool, far past it
    return 0;
}
''' % ROOT)
    exe = tmp_path / "rows"
    subprocess.run(["nvcc", "-std=c++17", "-arch=sm_100a", "--expt-relaxed-constexpr", "-o", str(exe), str(src)], check=True, capture_output=True, timeout=300)
    assert subprocess.run([str(exe)], timeout=60).returncode == 0
