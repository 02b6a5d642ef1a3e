"""The 4-bit KV cache through the C ABI against the oracle in 64 bits.

Bounds.  A stored element is rounded once: half a step of its type (eps / 2 of the value, 2^-25 below fp16's normal range), plus
2^-23 for the fp32 arithmetic before it.  An attention output adds what the probabilities and scores may be off: a probability
times a scale is rounded to fp16 (2^-11) and the exponential and the sums are fp32 (2^-19 together, generously); a score is a sum
of up to 256 fp32 terms, off by at most 2^-20 of the sum of their magnitudes (smag), which moves a probability by twice that in
relative terms (its own and the normalising sum).  Each times mag = sum_p w_p (code scale + |base|)."""
import ctypes

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
POISON = 0x7E00          # an fp16 NaN


def t(a):
    return torch.from_numpy(np.ascontiguousarray(a)).to(DEV)


def as64(x):
    return x.detach().cpu().double().numpy()


def half_step(dtype, ref):
    eps, tiny = (2.0 ** -10, 2.0 ** -25) if dtype == "f16" else (2.0 ** -7, 2.0 ** -134)
    return (eps / 2 * (1 + 2.0 ** -9) + 2.0 ** -23) * np.abs(ref) + tiny


def status(pkg, clear=True):
    v = ctypes.c_int(-1)
    st = torch.cuda.current_stream().cuda_stream
    pkg.lib().call("b200k_device_status", ctypes.addressof(v), st)
    if clear:
        pkg.lib().call("b200k_device_clear_status", st)
    return v.value


class Cache:
    """A 4-bit cache on the device, head-major or paged, filled with poison."""

    def __init__(self, batch, heads, d, g, max_len, block=0, seed=0):
        self.b, self.h, self.d, self.g, self.ml, self.block = batch, heads, d, g, max_len, block
        if block:
            self.per = -(-max_len // block)
            self.ml = self.per * block
            self.blocks = batch * self.per + 2
            self.table = np.random.default_rng(seed).permutation(self.blocks)[:batch * self.per].reshape(batch, self.per).astype(np.int32)
            self.dtable = t(self.table)
            lead = (self.blocks, heads, block)
        else:
            lead = (batch, heads, max_len)
        self.words = [torch.full(lead + (d // 8,), 0x5A5A5A5A, dtype=torch.int32, device=DEV) for _ in "kv"]
        self.params = [torch.full(lead + (d // g, 2), float("nan"), dtype=torch.float16, device=DEV) for _ in "kv"]

    @property
    def tensors(self):
        return self.words[0], self.params[0], self.words[1], self.params[1]

    def where(self, b, pos):
        """Index of [heads] rows of position pos of sequence b."""
        if self.block:
            return (int(self.table[b, pos // self.block]), slice(None), pos % self.block)
        return (b, slice(None), pos)

    def fill(self, k, v, lens, oracle):
        """Rows [b, heads, len, d] quantised by the oracle, put in place on the host."""
        for i, x in enumerate((k, v)):
            w, p = self.words[i].cpu().numpy(), self.params[i].cpu().numpy()
            for b, n in enumerate(lens):
                qw, qp = oracle.kv4_quantise(x[b][:, :n], self.g)
                for pos in range(n):
                    at = self.where(b, pos)
                    w[at], p[at] = qw[:, pos], qp[:, pos]
            self.words[i], self.params[i] = t(w), t(p)

    def rows(self, i, b, n):
        """(words [heads, n, ...], params) of the first n positions of sequence b, on the host."""
        w, p = self.words[i].cpu().numpy(), self.params[i].cpu().numpy()
        at = [self.where(b, pos) for pos in range(n)]
        if not n:
            return w[:0].reshape(self.h, 0, self.d // 8), p[:0].reshape(self.h, 0, self.d // self.g, 2)
        return np.stack([w[a] for a in at], 1), np.stack([p[a] for a in at], 1)

    def append(self, P, dtype, nk, nv, first, new, tokens, sk=None, sv=None):
        sk, sv = sk or self.h * self.d, sv or self.h * self.d
        if self.block:
            getattr(P, "kv_cache_append_paged_int4_" + dtype)(nk, nv, *self.tensors, self.dtable, first, new, self.h, self.d, self.g, self.block,
                                                              self.blocks, self.per, self.b, tokens, sk, sv)
        else:
            getattr(P, "kv_cache_append_hm_int4_" + dtype)(nk, nv, *self.tensors, first, new, self.h, self.d, self.g, self.ml, self.b, tokens, sk, sv)

    def read(self, P, dtype, first, lens, ko, vo):
        if self.block:
            getattr(P, "kv_cache_read_paged_int4_" + dtype)(*self.tensors, self.dtable, first, lens, ko, vo, self.h, self.d, self.g, self.block,
                                                            self.blocks, self.per, self.b, ko.shape[2])
        else:
            getattr(P, "kv_cache_read_hm_int4_" + dtype)(*self.tensors, first, lens, ko, vo, self.h, self.d, self.g, self.ml, self.b, ko.shape[2])

    def attend(self, P, dtype, q, lens, out, scale, ws=None, stream=None):
        name = "batched_decode_attention_%s_int4_%s" % ("paged" if self.block else "hm", dtype)
        tail = (scale,) if ws is None else (scale, ws, ws.numel() * ws.element_size())
        name += "" if ws is None else "_ws"
        if self.block:
            getattr(P, name)(q, *self.tensors, self.dtable, lens, out, self.b, q.shape[1], self.h, self.d, self.g, self.block, self.blocks, self.per,
                             *tail, stream=stream)
        else:
            getattr(P, name)(q, *self.tensors, lens, out, self.b, q.shape[1], self.h, self.d, self.g, self.ml, *tail, stream=stream)


def values(shape, dtype, seed, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * spread).to(TYPES[dtype]).to(DEV)


# ---- append ----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("heads,d,g", [(8, 128, 64), (2, 128, 128), (3, 128, 32), (1, 64, 64), (5, 32, 32), (2, 96, 32), (2, 160, 32), (1, 192, 64),
                                       (2, 224, 32), (2, 256, 128)])
@pytest.mark.parametrize("block,tokens", [(0, 1), (0, 7), (16, 1), (5, 19)])
def test_append_bits(P, pkg, oracle, dtype, heads, d, g, block, tokens):
    b = 3
    c = Cache(b, heads, d, g, 40, block, seed=d + tokens)
    nk, nv = values((b, tokens, heads, d), dtype, 1), values((b, tokens, heads, d), dtype, 2, 30.0)
    first = np.array([0, 13, c.ml - tokens], dtype=np.int32)
    want = [(w.cpu().numpy().copy(), p.cpu().numpy().view(np.uint16).copy()) for w, p in ((c.words[0], c.params[0]), (c.words[1], c.params[1]))]
    for i, x in enumerate((nk, nv)):
        qw, qp = oracle.kv4_quantise(as64(x), g)
        for s in range(b):
            for j in range(tokens):
                at = c.where(s, int(first[s]) + j)
                want[i][0][at], want[i][1][at] = qw[s, j], qp[s, j].view(np.uint16)
    status(pkg)
    c.append(P, dtype, nk, nv, t(first), None, tokens)
    assert status(pkg) == 0
    for i in range(2):
        assert (c.words[i].cpu().numpy() == want[i][0]).all()
        assert (c.params[i].cpu().numpy().view(np.uint16) == want[i][1]).all()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_append_special_values(P, oracle, dtype):
    """Constant groups, borders of two codes, tiny and huge values, infinities, NaN: each group on its own."""
    d, g, heads = 128, 32, 1
    rows = np.zeros((8, d), dtype=np.float64)
    rows[0] = -3.5
    rows[1, :64] = np.concatenate([[0, 15], np.arange(15) + 0.5, np.zeros(47)])
    rows[1, 64:] = 1000 + np.arange(64) % 7
    rows[2] = 6e-8 * (np.arange(d) % 5)                  # one subnormal step of fp16: the scale underflows to 0 or to one step
    rows[3, ::2], rows[3, 1::2] = 65504, -65504
    rows[4, 5], rows[4, 40], rows[4, 70], rows[4, 71] = np.inf, -np.inf, np.inf, -np.inf
    rows[5, 33], rows[5, 64], rows[5, 65] = np.nan, np.nan, np.inf
    rows[6] = -np.arange(d) * 0.25
    rows[7] = 1e-3 * np.where(np.arange(d) == 17, 1e6, np.arange(d))
    x = torch.from_numpy(rows).to(TYPES[dtype]).to(DEV).view(1, 8, heads, d)
    c = Cache(1, heads, d, g, 8)
    c.append(P, dtype, x, x.flip(1).contiguous(), t(np.zeros(1, np.int32)), None, 8)
    qw, qp = oracle.kv4_quantise(as64(x)[0], g)
    assert (c.words[0].cpu().numpy()[0].transpose(1, 0, 2) == qw).all()
    got = c.params[0].cpu().numpy()[0].transpose(1, 0, 2, 3)
    assert ((got == qp) | (np.isnan(got) & np.isnan(qp))).all()
    assert (c.words[1].cpu().numpy()[0].transpose(1, 0, 2) == qw[::-1]).all()
    ko, vo = (torch.empty(1, heads, 8, d, dtype=TYPES[dtype], device=DEV) for _ in "kv")
    c.read(P, dtype, None, t(np.array([8], np.int32)), ko, vo)
    back = as64(ko)[0, 0]
    assert np.isnan(back[5, 32:96]).all() and np.isfinite(np.delete(back, 5, 0)).all() and np.isfinite(back[5, :32]).all()


@pytest.mark.parametrize("block", [0, 8])
def test_append_padding_and_positions_outside(P, pkg, block):
    """Padding rows are not stored whatever they hold; rows outside the cache are skipped and reported."""
    heads, d, g, tokens = 2, 64, 32, 6
    c = Cache(4, heads, d, g, 16, block)
    nk, nv = values((4, tokens, heads, d), "f16", 3), values((4, tokens, heads, d), "f16", 4)
    new = np.array([0, 2, 6, -3], dtype=np.int32)
    for s in range(4):
        nk[s, max(new[s], 0):] = float("nan")
    first = np.array([3, 14, 0, 5], dtype=np.int32)
    before = [x.clone() for x in c.tensors]
    status(pkg)
    c.append(P, "f16", nk, nv, t(first), t(new), tokens)
    assert status(pkg) == 0
    changed = {(s, int(first[s]) + j) for s in range(4) for j in range(max(int(new[s]), 0))}
    for s in range(4):
        for pos in range(16):
            at = c.where(s, pos)
            same = torch.equal(c.words[0][at], before[0][at])
            assert same == ((s, pos) not in changed), (s, pos)
            assert torch.isfinite(c.params[0][at]).all().item() == ((s, pos) in changed)
    # positions before and behind the cache, a count above `tokens`
    c2 = Cache(4, heads, d, g, 16, block)
    nk = values((4, tokens, heads, d), "f16", 5)
    first = np.array([-2, 13, 2 ** 31 - 3, 4], dtype=np.int32)
    c2.append(P, "f16", nk, nk, t(first), t(np.array([6, 6, 6, 2 ** 31 - 1], np.int32)), tokens)
    assert status(pkg) & 4
    ok = {(0, 0), (0, 1), (0, 2), (0, 3), (1, 13), (1, 14), (1, 15)} | {(3, 4 + j) for j in range(6)}
    for s in range(4):
        for pos in range(16):
            assert torch.isfinite(c2.params[1][c2.where(s, pos)]).all().item() == ((s, pos) in ok), (s, pos)


def test_append_from_a_fused_row(P, oracle):
    """k and v as parts of one [batch, tokens, (hq + 2 hkv) d] tensor: the token stride is the fused row."""
    b, tokens, hq, hkv, d, g = 2, 3, 4, 2, 128, 64
    qkv = values((b, tokens, hq + 2 * hkv, d), "bf16", 6)
    st = (hq + 2 * hkv) * d
    flat = qkv.view(-1)
    c, c2 = Cache(b, hkv, d, g, 10), Cache(b, hkv, d, g, 10)
    first = t(np.array([1, 7], np.int32))
    c.append(P, "bf16", flat[hq * d:], flat[(hq + hkv) * d:], first, None, tokens, st, st)
    c2.append(P, "bf16", qkv[:, :, hq:hq + hkv].contiguous(), qkv[:, :, hq + hkv:].contiguous(), first, None, tokens)
    for x, y in zip(c.tensors, c2.tensors):
        assert torch.equal(x.view(torch.int16), y.view(torch.int16))


def test_bad_blocks_are_skipped_and_reported(P, pkg):
    c = Cache(2, 2, 64, 64, 12, 4)
    c.dtable[0, 1] = c.blocks
    c.dtable[1, 0] = -1
    x = values((2, 12, 2, 64), "f16", 8)
    status(pkg)
    c.append(P, "f16", x, x, t(np.zeros(2, np.int32)), None, 12)
    assert status(pkg) == 8
    ko = torch.full((2, 2, 12, 64), 7.0, dtype=torch.float16, device=DEV)
    vo = ko.clone()
    c.read(P, "f16", None, t(np.full(2, 12, np.int32)), ko, vo)
    assert status(pkg) == 8
    for o in (ko, vo):
        assert (o[0, :, 4:8] == 7).all() and (o[1, :, :4] == 7).all()
        assert torch.isfinite(o).all() and (o[0, :, :4] != 7).any() and (o[1, :, 4:] != 7).any()
    q, out = values((2, 4, 64), "f16", 9), torch.empty(2, 4, 64, dtype=torch.float16, device=DEV)
    c.attend(P, "f16", q, t(np.full(2, 12, np.int32)), out, 0.125)
    assert status(pkg) == 8 and torch.isfinite(out).all()
    c.attend(P, "f16", q, t(np.array([12, 4], np.int32)), out, 0.125)       # sequence 1 has nothing but the bad block: a zero row
    assert status(pkg) == 8 and (out[1] == 0).all() and (out[0] != 0).any()


# ---- read-back ---------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("heads,d,g,block", [(8, 128, 64, 0), (2, 128, 128, 16), (3, 128, 32, 7), (1, 64, 32, 0), (2, 96, 32, 4), (5, 32, 32, 0),
                                             (2, 256, 64, 16), (1, 224, 32, 0), (1, 256, 128, 0)])
def test_read_back(P, pkg, oracle, dtype, heads, d, g, block):
    b, ml = 4, 35
    c = Cache(b, heads, d, g, ml, block)
    lens = [0, 1, 35, 22]
    k, v = (as64(values((b, heads, ml, d), dtype, s, sp)) for s, sp in ((1, 1.0), (2, 1e-3)))
    c.fill(k, v, lens, oracle)
    for first, out_len in ((None, ml), ([0, 0, 30, 21], 9), ([5, 1, 34, 40], 3)):
        ko = torch.full((b, heads, out_len, d), 9.0, dtype=TYPES[dtype], device=DEV)
        vo = ko.clone()
        status(pkg)
        c.read(P, dtype, None if first is None else t(np.array(first, np.int32)), t(np.array(lens, np.int32)), ko, vo)
        assert status(pkg) == 0
        for i, o in enumerate((ko, vo)):
            for s in range(b):
                f = 0 if first is None else first[s]
                n = max(0, min(lens[s] - f, out_len))
                got = as64(o[s])
                assert (got[:, n:] == 9).all()                       # rows behind the context are left as they were
                if n:
                    w, p = c.rows(i, s, lens[s])
                    ref = oracle.kv4_values(w, p)[:, f:f + n]
                    assert (np.abs(got[:, :n] - ref) <= half_step(dtype, ref)).all()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("heads,d,g,block", [(8, 128, 64, 0), (8, 128, 32, 16), (2, 96, 32, 7), (1, 64, 64, 0), (3, 32, 32, 4), (4, 256, 128, 64),
                                             (1, 224, 32, 0)])
def test_read_back_of_many_rows(P, pkg, oracle, dtype, heads, d, g, block):
    """K and V by the same threads: rows of a large call against those of small ones, and a sample against the oracle."""
    b, rng = 4, np.random.default_rng(heads + d)
    n = 40000 // (b * heads) + 3                     # 8 b n heads threads are more than the machine holds at once
    c = big_cache(oracle, b, heads, d, g, n, 7, block)
    lens = t(np.array([n, n // 2 + 1, 0, 17], np.int32))
    part = n // 4 + 1

    def read(first, out_len):
        ko = torch.full((b, heads, out_len, d), 9.0, dtype=TYPES[dtype], device=DEV)
        vo = ko.clone()
        c.read(P, dtype, t(np.full(b, first, np.int32)), lens, ko, vo)
        return ko, vo
    status(pkg)
    whole = read(0, n)
    parts = [read(f, part) for f in range(0, n, part)]
    assert status(pkg) == 0
    for i, o in enumerate(whole):
        assert torch.equal(o.view(torch.int16), torch.cat([x[i] for x in parts], 2)[:, :, :n].contiguous().view(torch.int16))
        for s, m in enumerate(lens.tolist()):
            assert (o[s, :, m:] == 9).all()
            w, p = c.words[i].cpu().numpy(), c.params[i].cpu().numpy()
            for pos in rng.integers(0, m, 20 if m else 0):
                at = c.where(s, int(pos))
                ref = oracle.kv4_values(w[at], p[at])
                assert (np.abs(as64(o[s, :, pos]) - ref) <= half_step(dtype, ref)).all()


def test_read_lengths_and_starts_outside_are_reported(P, pkg, oracle):
    c = Cache(3, 1, 64, 64, 10)
    x = as64(values((3, 1, 10, 64), "f16", 1))
    c.fill(x, x, [10, 10, 10], oracle)
    ko = torch.full((3, 1, 12, 64), 9.0, dtype=torch.float16, device=DEV)
    vo = ko.clone()
    status(pkg)
    c.read(P, "f16", t(np.array([0, -2, 2 ** 31 - 1], np.int32)), t(np.array([2 ** 31 - 1, 4, -7], np.int32)), ko, vo)
    assert status(pkg) == 4
    assert (ko[0, :, :10] != 9).any() and (ko[0, :, 10:] == 9).all()
    assert (ko[1, :, :2] == 9).all() and (ko[1, :, 2:6] != 9).any() and (ko[1, :, 6:] == 9).all() and (ko[2] == 9).all()


# ---- RoPE + append -----------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("b,hq,hkv,d,g", [(5, 32, 8, 128, 64), (1, 4, 2, 64, 32), (3, 7, 1, 96, 32), (2, 4, 4, 256, 128), (4, 2, 1, 32, 32)])
def test_rope_append(P, pkg, oracle, dtype, b, hq, hkv, d, g):
    ml = 50
    rng = np.random.default_rng(d + b)
    pos = rng.permutation(ml)[:b].astype(np.int32)
    cos, sin = oracle.rope_tables(ml, d, 10000.0)
    qkv = values((b, hq + 2 * hkv, d), dtype, 11)
    c, c2 = Cache(b, hkv, d, g, ml), Cache(b, hkv, d, g, ml)
    q = torch.empty(b, hq, d, dtype=TYPES[dtype], device=DEV)
    status(pkg)
    getattr(P, "rope_kv_append_hm_int4_" + dtype)(qkv, t(cos), t(sin), t(pos), q, *c.tensors, hq, hkv, d, g, ml, b)
    assert status(pkg) == 0
    # fp32 products and sum, each rounded on its own; then one rounding to the type
    x = qkv[:, :hq + hkv].float()
    lo, hi = x[..., :d // 2], x[..., d // 2:]
    cc, ss = (t(a[pos])[:, None] for a in (cos, sin))
    rot = torch.cat((lo * cc - hi * ss, hi * cc + lo * ss), -1).to(TYPES[dtype])
    assert torch.equal(q, rot[:, :hq])
    c2.append(P, dtype, rot[:, hq:].contiguous(), qkv[:, hq + hkv:].contiguous(), t(pos), None, 1)
    for a, e in zip(c.tensors, c2.tensors):
        assert torch.equal(a.view(torch.int16), e.view(torch.int16))


def test_rope_append_positions_outside(P, pkg, oracle):
    b, hq, hkv, d, g, ml = 4, 4, 2, 128, 64, 9
    cos, sin = (t(a) for a in oracle.rope_tables(ml, d, 10000.0))
    qkv = values((b, hq + 2 * hkv, d), "f16", 12)
    c = Cache(b, hkv, d, g, ml)
    q = torch.empty(b, hq, d, dtype=torch.float16, device=DEV)
    status(pkg)
    P.rope_kv_append_hm_int4_f16(qkv, cos, sin, t(np.array([9, -1, 4, 2 ** 30], np.int32)), q, *c.tensors, hq, hkv, d, g, ml, b)
    assert status(pkg) == 4 and torch.isfinite(q).all()
    for s in range(b):
        for pos in range(ml):
            assert torch.isfinite(c.params[0][c.where(s, pos)]).all().item() == ((s, pos) == (2, 4))


# ---- attention -----------------------------------------------------------------------------------------------------------
def check_attention(oracle, c, q, lens, out, scale, dtype):
    for s, n in enumerate(lens):
        got = as64(out[s])
        if n <= 0:
            assert (got == 0).all()
            continue
        kw, kp = c.rows(0, s, n)
        vw, vp = c.rows(1, s, n)
        ref, mag, smag = oracle.kv4_decode_attention(as64(q[s]), kw, kp, vw, vp, scale)
        bound = half_step(dtype, ref) + (2.0 ** -11 + 2.0 ** -19 + 2 * 2.0 ** -20 * smag) * mag
        bad = ~(np.abs(got - ref) <= bound)
        assert not bad.any(), "seq %d len %d: %d of %d outside, worst %.3g against %.3g" % (
            s, n, bad.sum(), bad.size, np.abs(got - ref)[bad].max(), bound[bad].min())


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("hq,hkv,d,g,block,lens", [
    (32, 8, 128, 64, 0, [1, 15, 16, 17]),
    (32, 8, 128, 128, 16, [0, 333, 64, 1]),
    (16, 2, 128, 32, 0, [129, 500, 2]),
    (6, 2, 64, 64, 7, [31, 0, 100]),
    (4, 4, 64, 32, 0, [65, 33]),
    (10, 2, 256, 128, 0, [77, 256]),
    (7, 1, 256, 32, 16, [40]),
    (32, 2, 128, 64, 0, [200]),          # groups of 16 q heads
    (9, 1, 96, 32, 0, [55, 70]),
    (3, 3, 32, 32, 4, [10, 129]),
    (8, 2, 160, 32, 0, [130]),
    (4, 1, 192, 64, 0, [130, 5]),
    (2, 1, 224, 32, 16, [50]),
])
def test_attention(P, pkg, oracle, dtype, hq, hkv, d, g, block, lens):
    b, ml = len(lens), max(lens) + 3
    c = Cache(b, hkv, d, g, ml, block, seed=hq)
    k, v = as64(values((b, hkv, ml, d), dtype, 21)), as64(values((b, hkv, ml, d), dtype, 22))
    c.fill(k, v, lens, oracle)            # rows behind a context stay poisoned: NaN scales
    q = values((b, hq, d), dtype, 23)
    out = torch.full((b, hq, d), float("nan"), dtype=TYPES[dtype], device=DEV)
    scale = d ** -0.5
    status(pkg)
    c.attend(P, dtype, q, t(np.array(lens, np.int32)), out, scale)
    assert status(pkg) == 0
    check_attention(oracle, c, q, lens, out, scale, dtype)
    again = torch.empty_like(out)
    c.attend(P, dtype, q, t(np.array(lens, np.int32)), again, scale)
    assert torch.equal(out, again), "two runs differ"


@pytest.mark.parametrize("kspread,vspread,qspread,scale", [(1.0, 1e-4, 1.0, 0.088), (30.0, 1000.0, 1.0, 0.088), (1e-3, 1.0, 1e-3, 0.088), (1.0, 1.0, 900.0, 0.088),
                                                           (1.0, 1.0, 1.0, -0.1), (1.0, 1.0, 1.0, 0.0), (0.0, 1.0, 1.0, 1.0), (1.0, 0.0, 0.0, 1.0)])
def test_attention_ranges(P, oracle, kspread, vspread, qspread, scale):
    """Tiny, huge and constant keys, values and queries, peaked and flat softmaxes, a negative and a zero scale."""
    b, hq, hkv, d, g, n = 2, 8, 2, 128, 64, 300
    c = Cache(b, hkv, d, g, n)
    k, v = as64(values((b, hkv, n, d), "f16", 31, kspread)), as64(values((b, hkv, n, d), "f16", 32, vspread))
    c.fill(k, v, [n, n - 7], oracle)
    q = values((b, hq, d), "f16", 33, qspread)
    out = torch.empty((b, hq, d), dtype=torch.float16, device=DEV)
    c.attend(P, "f16", q, t(np.array([n, n - 7], np.int32)), out, scale)
    check_attention(oracle, c, q, [n, n - 7], out, scale, "f16")


def test_attention_value_scales_that_grow(P, oracle):
    """Values whose magnitude grows along the context by 2^20, then falls: no product may over- or underflow on the way."""
    hq, hkv, d, g, n = 4, 1, 128, 64, 400
    ramp = 2.0 ** (np.concatenate([np.arange(n // 2), np.arange(n - n // 2)[::-1]]) / 10 - 10)
    k = as64(values((1, hkv, n, d), "f16", 41))
    v = as64((values((1, hkv, n, d), "f16", 42).double() * t(ramp)[None, None, :, None]).half())
    c = Cache(1, hkv, d, g, n)
    c.fill(k, v, [n], oracle)
    q = values((1, hq, d), "f16", 43, 0.1)
    out = torch.empty((1, hq, d), dtype=torch.float16, device=DEV)
    for m in (n, 30, 200):
        c.attend(P, "f16", q, t(np.array([m], np.int32)), out, 0.088)
        check_attention(oracle, c, q, [m], out, 0.088, "f16")


def test_attention_growing_scores(P, oracle):
    """Scores that climb by hundreds along the context: the running maximum moves in every tile."""
    hq, hkv, d, g, n = 8, 1, 64, 32, 260
    k = np.zeros((1, hkv, n, d))
    k[0, 0] = np.linspace(-40, 40, n)[:, None]
    k = as64(torch.from_numpy(k).half())
    v = as64(values((1, hkv, n, d), "f16", 52))
    c = Cache(1, hkv, d, g, n)
    c.fill(k, v, [n], oracle)
    q = torch.ones(1, hq, d, dtype=torch.float16, device=DEV)
    q[0, 1::2] = -1
    out = torch.empty((1, hq, d), dtype=torch.float16, device=DEV)
    c.attend(P, "f16", q, t(np.array([n], np.int32)), out, 0.125)
    check_attention(oracle, c, q, [n], out, 0.125, "f16")


def test_attention_nan_stays_with_its_head(P, oracle):
    """A NaN key within the context makes the heads that read it NaN and no other."""
    hq, hkv, d, g, n = 8, 2, 128, 64, 50
    k, v = as64(values((2, hkv, n, d), "f16", 61)), as64(values((2, hkv, n, d), "f16", 62))
    k[0, 1, 20, 3] = np.nan
    c = Cache(2, hkv, d, g, n)
    c.fill(k, v, [n, n], oracle)
    q = values((2, hq, d), "f16", 63)
    out = torch.empty((2, hq, d), dtype=torch.float16, device=DEV)
    c.attend(P, "f16", q, t(np.array([n, n], np.int32)), out, 0.088)
    assert torch.isnan(out[0, 4:]).all() and torch.isfinite(out[0, :4]).all() and torch.isfinite(out[1]).all()


@pytest.mark.parametrize("d,g", [(128, 32), (256, 64)])
@pytest.mark.parametrize("kspread,vspread,kmean,vmean,scale", [
    (1.0, 1.0, 0.0, 0.0, 0.09), (1.0, 1e-4, 0.0, 0.0, 0.09), (30.0, 1000.0, 0.0, 0.0, 0.02), (1.0, 1.0, 50.0, -100.0, 0.09), (1.0, 8000.0, 0.0, 20000.0, 0.09),
    (1.0, 0.0, 0.0, 3.0, 0.09), (0.0, 1.0, 2.0, 0.0, 1.0), (1.0, 1.0, 0.0, 0.0, -0.1), (1.0, 1.0, 0.0, 0.0, 0.0)])
def test_attention_with_four_groups(P, oracle, d, g, kspread, vspread, kmean, vmean, scale):
    """Their bases go through matrix instructions: far off-centre, tiny, huge and constant keys and values."""
    b, hq, hkv, n = 3, 10, 2, 420
    lens = [n, n - 7, 5]
    c = Cache(b, hkv, d, g, n)
    k = as64((values((b, hkv, n, d), "f16", 31, kspread).float() + kmean).half())
    v = as64((values((b, hkv, n, d), "f16", 32, vspread).float() + vmean).clamp(-60000, 60000).half())
    c.fill(k, v, lens, oracle)
    q = values((b, hq, d), "f16", 33)
    out = torch.empty((b, hq, d), dtype=torch.float16, device=DEV)
    c.attend(P, "f16", q, t(np.array(lens, np.int32)), out, scale)
    check_attention(oracle, c, q, lens, out, scale, "f16")


@pytest.mark.parametrize("d,g", [(128, 32), (128, 64)])
@pytest.mark.parametrize("vspread,vmean", [(1.0, 0.0), (8000.0, 20000.0), (1e-3, 5.0)])
def test_one_position_over_many_small_ones(P, oracle, d, g, vspread, vmean):
    """Probabilities 2^-16.6 of the largest, whose sum counts: none may vanish in 16 bits.  600 contexts, so that a warp has 512
    positions of one; the value scales grow on the way."""
    b, n = 600, 2000
    c = Cache(b, 1, d, g, n)
    gen = torch.Generator(device=DEV).manual_seed(5)
    k = torch.zeros(b, n, 1, d, dtype=torch.float16, device=DEV)
    k[:, 0, 0, :] = 11.5 / d
    v = (torch.randn(b, n, 1, d, device=DEV, generator=gen) * vspread * torch.linspace(0.01, 1.0, n, device=DEV)[None, :, None, None] + vmean).half()
    c.append(P, "f16", k, v, t(np.zeros(b, np.int32)), None, n)
    q = torch.ones(b, 2, d, dtype=torch.float16, device=DEV)
    out = torch.empty_like(q)
    c.attend(P, "f16", q, t(np.full(b, n, np.int32)), out, 1.0)
    for s in (0, 311, 599):
        (kw, kp), (vw, vp) = c.rows(0, s, n), c.rows(1, s, n)
        ref, mag, smag = oracle.kv4_decode_attention(as64(q[s]), kw, kp, vw, vp, 1.0)
        bound = half_step("f16", ref) + (2.0 ** -11 + 2.0 ** -19 + 2 * 2.0 ** -20 * smag) * mag
        assert (np.abs(as64(out[s]) - ref) <= bound).all()


@pytest.mark.parametrize("d,g", [(128, 32), (128, 64), (256, 64), (96, 32), (64, 32)])
def test_value_nan_stays_with_its_group(P, oracle, d, g):
    hq, hkv, n = 4, 1, 90
    k, v = as64(values((1, hkv, n, d), "f16", 61)), as64(values((1, hkv, n, d), "f16", 62))
    v[0, 0, 70, 40] = np.nan
    c = Cache(1, hkv, d, g, n)
    c.fill(k, v, [n], oracle)
    q = values((1, hq, d), "f16", 63)
    out = torch.empty((1, hq, d), dtype=torch.float16, device=DEV)
    c.attend(P, "f16", q, t(np.array([n], np.int32)), out, 0.088)
    bad = torch.zeros(d, dtype=torch.bool, device=DEV)
    bad[40 // g * g:40 // g * g + g] = True
    assert torch.isnan(out[..., bad]).all() and torch.isfinite(out[..., ~bad]).all()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("hq,hkv,d,g,block", [(3, 3, 32, 32, 4), (4, 4, 64, 32, 0), (6, 2, 64, 64, 7), (9, 1, 96, 32, 0), (16, 2, 128, 32, 0), (32, 8, 128, 64, 16),
                                              (32, 2, 128, 128, 0), (8, 2, 160, 32, 0), (4, 1, 192, 64, 0), (4, 2, 192, 32, 32), (2, 1, 224, 32, 16),
                                              (7, 1, 256, 32, 16), (4, 1, 256, 64, 0), (10, 2, 256, 128, 0)])
def test_attention_cut_and_whole_contexts(P, oracle, dtype, hq, hkv, d, g, block):
    """Every shape with contexts that several CTAs share and, in a call of their own, with ones that one CTA has."""
    c = Cache(3, hkv, d, g, 700, block, seed=d)
    lens = [700, 385, 1]
    k, v = as64(values((3, hkv, 700, d), dtype, 24)), as64(values((3, hkv, 700, d), dtype, 25))
    c.fill(k, v, lens, oracle)
    q = values((3, hq, d), dtype, 26)
    for now in (lens, [256, 129, 1]):
        out = torch.full((3, hq, d), float("nan"), dtype=TYPES[dtype], device=DEV)
        c.attend(P, dtype, q, t(np.array(now, np.int32)), out, d ** -0.5)
        check_attention(oracle, c, q, now, out, d ** -0.5, dtype)


@pytest.mark.parametrize("hq,hkv,d,g", [(8, 2, 128, 64), (4, 4, 128, 128), (3, 1, 64, 64), (8, 2, 96, 32), (6, 3, 256, 128)])
def test_attention_of_few_heads_loses_nothing_but_the_output_rounding(P, oracle, hq, hkv, d, g):
    """Up to 4 q heads a kv head, fp16: 22 bits of a probability times a scale count (2^-22), so of the general bound's 2^-11 there
    remains what the exponential and the fp32 sums are off (2^-19, and 2^-19 for what the tensor cores cut off)."""
    b, n = 2, 420
    c = Cache(b, hkv, d, g, n)
    lens = [n, n - 130]
    k, v = as64(values((b, hkv, n, d), "f16", 71)), as64(values((b, hkv, n, d), "f16", 72))
    c.fill(k, v, lens, oracle)
    q = values((b, hq, d), "f16", 73)
    out = torch.empty((b, hq, d), dtype=torch.float16, device=DEV)
    c.attend(P, "f16", q, t(np.array(lens, np.int32)), out, d ** -0.5)
    for s, m in enumerate(lens):
        (kw, kp), (vw, vp) = c.rows(0, s, m), c.rows(1, s, m)
        ref, mag, smag = oracle.kv4_decode_attention(as64(q[s]), kw, kp, vw, vp, d ** -0.5)
        bound = half_step("f16", ref) + (2.0 ** -22 + 2.0 ** -18 + 2 * 2.0 ** -20 * smag) * mag
        assert (np.abs(as64(out[s]) - ref) <= bound).all()


def big_cache(oracle, b, hkv, d, g, n, seed, block=0):
    """A long cache: random words and params straight on the device."""
    c = Cache(b, hkv, d, g, n, block, seed)
    gen = torch.Generator(device=DEV).manual_seed(seed)
    for i in range(2):
        c.words[i].random_(-2 ** 31, 2 ** 31 - 1, generator=gen)
        c.params[i][..., 0] = torch.rand(c.params[i].shape[:-1], device=DEV, generator=gen) * 0.2 + 0.2
        c.params[i][..., 1] = -torch.rand(c.params[i].shape[:-1], device=DEV, generator=gen) - 2
    return c


@pytest.mark.parametrize("b,hq,hkv,d,g,block,lens", [
    (1, 32, 8, 128, 64, 0, [20011]),
    (3, 8, 2, 128, 128, 64, [9000, 0, 4097]),
    (40, 8, 1, 64, 32, 0, None),
    (2, 16, 1, 256, 64, 16, [5000, 12]),
    (200, 8, 4, 128, 64, 0, None),        # more contexts than CTAs: a CTA goes through several, cut at both ends
    (90, 16, 8, 64, 64, 16, None),
    (1, 4, 1, 64, 32, 0, [80001]),        # one context over every CTA: three rounds of joining
])
def test_attention_long_and_ragged(P, oracle, b, hq, hkv, d, g, block, lens):
    rng = np.random.default_rng(b)
    lens = lens or [int(x) for x in rng.integers(0, 1500 if b < 50 else 400, b)]
    c = big_cache(oracle, b, hkv, d, g, max(lens), 70 + b, block)
    q = values((b, hq, d), "f16", 71)
    out = torch.full((b, hq, d), float("nan"), dtype=torch.float16, device=DEV)
    c.attend(P, "f16", q, t(np.array(lens, np.int32)), out, d ** -0.5)
    check_attention(oracle, c, q, lens, out, d ** -0.5, "f16")


def test_attention_length_beyond_the_cache_is_clamped_and_reported(P, pkg, oracle):
    c = big_cache(oracle, 3, 2, 128, 64, 700, 5)
    q = values((3, 8, 128), "f16", 72)
    want, got = (torch.empty((3, 8, 128), dtype=torch.float16, device=DEV) for _ in range(2))
    status(pkg)
    c.attend(P, "f16", q, t(np.array([700, 37, 700], np.int32)), want, 0.088)
    assert status(pkg) == 0
    c.attend(P, "f16", q, t(np.array([701, 37, 2 ** 31 - 1], np.int32)), got, 0.088)
    assert status(pkg) == 4 and torch.equal(want, got)
    c.attend(P, "f16", q, t(np.array([700, 37, -(2 ** 31)], np.int32)), got, 0.088)
    assert status(pkg) == 0 and torch.equal(want[:2], got[:2]) and (got[2] == 0).all()


def test_tables_that_share_blocks(P, oracle):
    """Sequences with a common prefix read the same blocks; a table entry behind a context may be anything."""
    hq, hkv, d, g, block, n = 8, 2, 128, 64, 16, 100
    c = Cache(3, hkv, d, g, n, block)
    k, v = (as64(values((1, hkv, n, d), "f16", s)).repeat(3, 0) for s in (91, 92))
    c.table[1:] = c.table[0]
    c.dtable = t(c.table)
    c.fill(k, v, [n, n, n], oracle)
    q = values((1, hq, d), "f16", 93).repeat(3, 1, 1)
    out = torch.empty_like(q)
    lens = [n, 33, 48]
    bad = c.table.copy()
    bad[1, 3:], bad[2, 3:] = 2 ** 31 - 1, -5
    c.dtable = t(bad)
    c.attend(P, "f16", q, t(np.array(lens, np.int32)), out, 0.088)
    check_attention(oracle, c, q, lens, out, 0.088, "f16")


def test_attention_offsets_beyond_32_bits(P, oracle):
    """The last sequence of a cache of 9 x 2^24 rows of 64 dims: its codes start beyond 4 GiB, its units beyond 2^31."""
    b, n, d, g = 9, 1 << 24, 64, 64
    lead = (b, 1, n)
    c = Cache.__new__(Cache)
    c.b, c.h, c.d, c.g, c.ml, c.block = b, 1, d, g, n, 0
    c.words = [torch.zeros(lead + (d // 8,), dtype=torch.int32, device=DEV) for _ in "kv"]
    c.params = [torch.zeros(lead + (1, 2), dtype=torch.float16, device=DEV) for _ in "kv"]
    x, y = values((b, 3, 1, d), "f16", 81), values((b, 3, 1, d), "f16", 82)
    first = t(np.array([0] * 8 + [n - 3], np.int32))
    c.append(P, "f16", x, y, first, None, 3)
    qw, qp = oracle.kv4_quantise(as64(x)[8], g)
    assert (c.words[0][8, 0, n - 3:].cpu().numpy() == qw[:, 0]).all()
    assert (c.params[0][8, 0, n - 3:].cpu().numpy() == qp[:, 0]).all()
    ko, vo = (torch.zeros(b, 1, 3, d, dtype=torch.float16, device=DEV) for _ in "kv")
    c.read(P, "f16", first, t(np.array([3] * 8 + [n], np.int32)), ko, vo)
    for i, (o, z) in enumerate(((ko, x), (vo, y))):
        ref = oracle.kv4_values(*oracle.kv4_quantise(as64(z)[:, :, 0], g))
        assert (np.abs(as64(o)[:, 0] - ref) <= half_step("f16", ref)).all()
    # a context that ends in the cache's last rows: everything before is zero keys and values of equal weight
    q = values((b, 2, d), "f16", 83)
    out = torch.empty((b, 2, d), dtype=torch.float16, device=DEV)
    c.attend(P, "f16", q, t(np.array([3] * 8 + [n], np.int32)), out, 60.0)
    v8 = oracle.kv4_values(*oracle.kv4_quantise(as64(y)[8], g))[:, 0]
    k8 = oracle.kv4_values(qw, qp)[:, 0]
    for h in range(2):
        z = np.concatenate([k8 @ as64(q[8, h]) * 60.0, [0.0]])
        w = np.exp(z - z.max())
        w[3] *= n - 3
        ref = (w[:3] / w.sum()) @ v8
        mag = (w[:3] / w.sum()) @ np.abs(oracle.kv4_values(qw, np.abs(qp))[:, 0])
        smag = 60.0 * np.max(oracle.kv4_values(qw, np.abs(qp))[:, 0] @ np.abs(as64(q[8, h])))
        assert (np.abs(as64(out[8, h]) - ref) <= half_step("f16", ref) + (2.0 ** -10 + 2.0 ** -18 + 2.0 ** -19 * smag) * mag).all()


# ---- streams, graphs, workspaces ---------------------------------------------------------------------------------------
def test_two_streams_with_a_workspace_each(P, pkg, oracle):
    cs = [big_cache(oracle, 1, 8, 128, 64, 6000, s) for s in (1, 2)]
    qs = [values((1, 32, 128), "f16", s) for s in (3, 4)]
    lens = t(np.array([6000], np.int32))
    nbytes = pkg.lib().call("b200k_attention_int4_workspace_bytes", 1, 32, 8, 128)
    want = [torch.empty((1, 32, 128), dtype=torch.float16, device=DEV) for _ in range(2)]
    for c, q, o in zip(cs, qs, want):
        c.attend(P, "f16", q, lens, o, 0.088)
    ws = [torch.zeros(nbytes, dtype=torch.uint8, device=DEV) for _ in range(2)]
    got = [torch.empty((1, 32, 128), dtype=torch.float16, device=DEV) for _ in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(10):
        for c, q, o, w, s in zip(cs, qs, got, ws, streams):
            c.attend(P, "f16", q, lens, o, 0.088, ws=w, stream=s.cuda_stream)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    assert all(int(w[:128 * 1024].count_nonzero()) == 0 for w in ws)          # counters and status word left at zero


def test_two_graphs_share_a_workspace(P, pkg, oracle):
    """Two captured calls of different shapes on one workspace, replayed in turn: every launch finds the counters at zero."""
    cs = [big_cache(oracle, 1, 8, 128, 64, 9000, 1), big_cache(oracle, 130, 5, 64, 32, 300, 2)]
    qs = [values((1, 32, 128), "f16", 3), values((130, 10, 64), "bf16", 4)]
    lens = [t(np.array([9000], np.int32)), t(np.random.default_rng(3).integers(0, 301, 130).astype(np.int32))]
    kinds, scale = ["f16", "bf16"], 0.1
    ws = torch.zeros(pkg.lib().call("b200k_attention_int4_workspace_bytes", 1, 32, 8, 128), dtype=torch.uint8, device=DEV)
    want, got, graphs = [], [], []
    for c, q, n, k in zip(cs, qs, lens, kinds):
        want.append(torch.empty_like(q))
        got.append(torch.empty_like(q))
        c.attend(P, k, q, n, want[-1], scale)
    torch.cuda.synchronize()
    for c, q, n, k, o in zip(cs, qs, lens, kinds, got):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            c.attend(P, k, q, n, o, scale, ws=ws)
    for i in (0, 1, 1, 0, 0, 1):
        got[i].zero_()
        graphs[i].replay()
        torch.cuda.synchronize()
        assert torch.equal(got[i], want[i])
    assert int(ws[:128 * 1024].count_nonzero()) == 0


def test_captured_graph_follows_the_lengths(P, oracle):
    """One captured append + attention, replayed while positions, lengths and inputs move on the device."""
    b, hq, hkv, d, g, ml = 3, 8, 2, 128, 64, 900
    c, e = big_cache(oracle, b, hkv, d, g, ml, 9), big_cache(oracle, b, hkv, d, g, ml, 9)
    nk, nv, q = values((b, 1, hkv, d), "f16", 1), values((b, 1, hkv, d), "f16", 2), values((b, hq, d), "f16", 3)
    pos, lens = t(np.array([5, 0, 700], np.int32)), t(np.array([6, 1, 701], np.int32))
    out, want = (torch.empty((b, hq, d), dtype=torch.float16, device=DEV) for _ in range(2))

    def step(cache, o):
        cache.append(P, "f16", nk, nv, pos, None, 1)
        cache.attend(P, "f16", q, lens, o, 0.088)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(e, want)                      # first-use set-up happens outside the capture
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(c, out)
    for i, p in enumerate(([5, 0, 700], [6, 1, 701], [300, 898, 3])):
        pos.copy_(t(np.array(p, np.int32)))
        lens.copy_(pos + 1)
        for x, s in ((nk, 10), (nv, 20), (q, 30)):
            x.copy_(values(x.shape, "f16", s + i))
        graph.replay()
        step(e, want)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        assert all(torch.equal(a.view(torch.int16), z.view(torch.int16)) for a, z in zip(c.tensors, e.tensors))


def test_chunked_prefill_then_decode(P, pkg, oracle):
    """The operators as a server runs them: a prompt in two chunks (append, read back, prefill attention), then decode steps
    (RoPE + append, attention), against the same steps in 64 bits on the rows as stored."""
    hq, hkv, d, g, ml, block = 8, 2, 128, 64, 96, 16
    scale = d ** -0.5
    for blk in (0, block):
        c = Cache(1, hkv, d, g, ml, blk)
        prompt = 50
        k, v, q = values((1, prompt, hkv, d), "f16", 91), values((1, prompt, hkv, d), "f16", 92), values((1, hq, prompt, d), "f16", 93)
        done = 0
        for n in (33, 17):
            c.append(P, "f16", k[:, done:done + n].contiguous(), v[:, done:done + n].contiguous(), t(np.array([done], np.int32)), None, n)
            total = done + n
            ko, vo = (torch.zeros(1, hkv, total, d, dtype=torch.float16, device=DEV) for _ in "kv")
            c.read(P, "f16", None, t(np.array([total], np.int32)), ko, vo)
            out = torch.empty(1, hq, n, d, dtype=torch.float16, device=DEV)
            P.flash_attn_full_f16(q[:, :, done:total].contiguous(), ko, vo, out, 1, hq, hkv, n, total, d, done, scale)
            ref = oracle.flash_attn_full(as64(q[:, :, done:total]).astype(np.float32), as64(ko).astype(np.float32), as64(vo).astype(np.float32), done, scale)
            assert np.abs(as64(out) - ref).max() <= 1e-2 + 1e-2 * np.abs(ref).max()
            done = total
        if blk:
            continue
        cos, sin = (t(a) for a in oracle.rope_tables(ml, d, 10000.0))
        for step in range(4):
            qkv = values((1, (hq + 2 * hkv) * d), "f16", 100 + step)
            qr, out = (torch.empty(1, hq, d, dtype=torch.float16, device=DEV) for _ in range(2))
            P.rope_kv_append_hm_int4_f16(qkv, cos, sin, t(np.array([done], np.int32)), qr, *c.tensors, hq, hkv, d, g, ml, 1)
            done += 1
            c.attend(P, "f16", qr, t(np.array([done], np.int32)), out, scale)
            check_attention(oracle, c, qr, [done], out, scale, "f16")


@pytest.mark.parametrize("use_graph", [False, True])
@pytest.mark.parametrize("awq", [False, True])
def test_decode_layer_over_a_4_bit_cache(pkg, P, oracle, use_graph, awq):
    """The layer's steps with the 4-bit cache, against the same entry points called one by one (bit for bit), and a switch back to
    the fp16 cache."""
    rng = np.random.default_rng(5)
    B, H, hq, hkv, d, I, G, ml, kg = 3, 256, 4, 2, 128, 384, 128, 40, 64

    def weight(k, n):
        sc = rng.uniform(0.002, 0.02, (k // G, n)).astype(np.float16)
        if awq:
            return (t(oracle.pack_awq(rng.integers(0, 16, (k, n), dtype=np.int32))), t(sc), t(oracle.pack_awq(rng.integers(0, 16, (k // G, n), dtype=np.int32))))
        return (t(oracle.pack_gptq_qweight(rng.integers(1, 16, (k, n), dtype=np.int32))), t(sc), t(np.full((k // G, n // 8), 0x77777777, dtype=np.int32)))
    w = {"qkv": weight(H, (hq + 2 * hkv) * d), "o": weight(hq * d, H), "gate_up": weight(H, 2 * I), "down": weight(I, H)}
    ln1, ln2 = (t(rng.uniform(0.5, 1.5, H).astype(np.float16)) for _ in range(2))
    cos, sin = (t(a) for a in oracle.rope_tables(ml, d, 500000.0))
    fmt = "awq" if awq else "gptq"
    layer = pkg.DecodeLayer(pkg.LayerShape(H, hq, hkv, d, I, G, 1e-5), w, ln1, ln2, cos, sin, max_batch=4, max_len=ml, fmt=fmt, use_graph=use_graph,
                            kv_group_size=kg)
    c = Cache(4, hkv, d, kg, ml)
    c.words, c.params = [torch.zeros_like(x) for x in c.words], [torch.zeros_like(x) for x in c.params]
    gemm = P.awq_gemm if awq else P.gptq_gemm
    hid, pos, out = torch.empty(B, H, dtype=torch.float16, device=DEV), torch.empty(B, dtype=torch.int32, device=DEV), torch.empty(B, H, dtype=torch.float16, device=DEV)
    for p in ([5, 0, 38], [6, 1, 39], [7, 2, 3]):               # the first step captures, the others replay
        hid.copy_(torch.from_numpy(rng.standard_normal((B, H)).astype(np.float16)))
        pos.copy_(torch.tensor(p, dtype=torch.int32))
        layer.forward(hid, pos, out=out)
        n1, n2, h1, want = (torch.empty_like(hid) for _ in range(4))
        P.rms_norm_f16(hid, ln1, n1, H, 1.0 / H, 1e-5, B)
        qkv = gemm(n1, *w["qkv"], G)
        q, att = (torch.empty(B, hq, d, dtype=torch.float16, device=DEV) for _ in range(2))
        P.rope_kv_append_hm_int4_f16(qkv, cos, sin, pos, q, *c.tensors, hq, hkv, d, kg, ml, B)
        P.batched_decode_attention_hm_int4_f16(q, *c.tensors, pos + 1, att, B, hq, hkv, d, kg, ml, 1.0 / float(np.sqrt(d)))
        o = gemm(att.view(B, hq * d), *w["o"], G)
        P.fused_add_rms_norm_f16(o, hid, ln2, n2, h1, H, 1.0 / H, 1e-5, B)
        gu = gemm(n2, *w["gate_up"], G)
        act = torch.empty(B, I, dtype=torch.float16, device=DEV)
        P.fused_silu_mul_interleaved_f16(gu, act, I, B * I)
        dn = gemm(act, *w["down"], G)
        P.residual_add_f16(h1, dn, want, B * H)
        torch.cuda.synchronize()
        assert torch.isfinite(out).all() and torch.equal(out, want)
        for a, b in zip((*layer.k_cache, *layer.v_cache), c.tensors):
            assert torch.equal(a, b)
    half = [torch.zeros(4, hkv, ml, d, dtype=torch.float16, device=DEV) for _ in "kv"]
    pkg.lib().call("b200k_layer_set_kv_cache", layer.handle, *half)
    before = [x.clone() for x in (*layer.k_cache, *layer.v_cache)]
    layer.forward(hid, pos, out=out)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(before, (*layer.k_cache, *layer.v_cache)))
    layer.close()
