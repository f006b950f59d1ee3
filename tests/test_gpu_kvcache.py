"""The paged-cache operators (kvcache.py, include/s2d_cache.h) against plain 64-bit forms.

Unused pages, the rows of a page past a sequence's length, and the mass and positions of free slots are NaN or nonsense in
every case: nothing may read them into a result.
"""
import math

import numpy as np
import pytest

import kvcache_reference as ref

pytestmark = pytest.mark.gpu

PAGE = 64
# Half a step of each type relative to a value; f32 results are held to the attention tests' 2e-5 of the largest value.
HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
F32_TOL = 2e-5


@pytest.fixture(scope="module")
def torch():
    import torch
    return torch


def act_dtype(torch, ty):
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[ty]


def rounded(torch, x, dtype):
    """float64 numpy of x rounded to dtype, and the tensor."""
    t = torch.from_numpy(np.asarray(x, np.float32)).to(dtype)
    return t.double().numpy(), t.cuda()


class Case:
    """A cache of random pages: k64 / v64 the values in float64 (NaN outside the sequences), c the PagedKvCache."""

    def __init__(self, torch, ty, H, G, D, lengths, tokens=None, prefix_len=0, extra_pages=3, layered=False, spare=0, seed=0, pad=0,
                 k_scale=1.0):
        from fish_s2pro_b200 import PagedKvCache
        rng = np.random.default_rng(seed + 17 * D + H)
        self.torch, self.ty, self.H, self.G, self.D = torch, ty, H, G, D
        self.kv = torch.bfloat16 if ty == "bf16" else torch.float16
        B = len(lengths)
        per = max(1, -(-max(max(lengths), 1) // PAGE)) + spare
        n_prefix = -(-prefix_len // PAGE)
        n_pages = B * per + n_prefix + extra_pages
        ids = rng.permutation(n_pages)
        self.table, self.prefix = ids[: B * per].reshape(B, per), ids[B * per: B * per + n_prefix]
        pool = np.full((2, n_pages, G, PAGE, D), np.nan, np.float32)
        for i in range(2):
            for b in range(B):
                for j in range(0, lengths[b], PAGE):
                    m = min(PAGE, lengths[b] - j)
                    pool[i, self.table[b, j // PAGE], :, :m] = rng.standard_normal((G, m, D)) * (k_scale if i == 0 else 1.0)
            for j in range(0, prefix_len, PAGE):
                m = min(PAGE, prefix_len - j)
                pool[i, self.prefix[j // PAGE], :, :m] = rng.standard_normal((G, m, D)) * (k_scale if i == 0 else 1.0)
        (self.k64, k), (self.v64, v) = rounded(torch, pool[0], self.kv), rounded(torch, pool[1], self.kv)
        if layered:  # layer 1 of a pool laid out [page][layer][K | V][head][64][D]
            big = torch.full((n_pages, 3, 2, G, PAGE, D), float("nan"), dtype=self.kv, device="cuda")
            big[:, 1, 0], big[:, 1, 1] = k, v
            k, v = big[:, 1, 0], big[:, 1, 1]
        self.lengths = np.asarray(lengths, np.int32)
        self.scale = 1 / math.sqrt(D)
        slots = per * PAGE
        self.mass0 = np.full((B, G, slots), np.nan, np.float32)
        for b in range(B):
            self.mass0[b, :, : lengths[b]] = rng.random((G, lengths[b]))
        self.pos0 = np.broadcast_to(np.arange(slots, dtype=np.int32), (B, G, slots)).copy()
        self.mass, self.positions = (torch.from_numpy(x.copy()).cuda() for x in (self.mass0, self.pos0))
        self.ints = lambda x: torch.from_numpy(np.asarray(x, np.int32)).cuda()
        self.c = PagedKvCache(k, v, self.ints(self.table), self.ints(lengths), positions=self.positions, mass=self.mass)
        self.tokens = tokens
        counts = [1] * B if tokens is None else tokens
        self.starts = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        T = int(self.starts[-1]) + pad
        self.q64, self.q = rounded(torch, rng.standard_normal((T, H, D)) * 2.0, act_dtype(torch, ty))
        self.q_start = None if tokens is None else self.ints(self.starts)
        self.prefix_len = prefix_len
        self.prefix_pages = self.ints(self.prefix) if prefix_len else None

    def attend(self, **kw):
        return self.c.attention(self.q, q_start=self.q_start, prefix_pages=self.prefix_pages, prefix_len=self.prefix_len,
                                return_lse=True, **kw)

    def expected(self):
        return ref.attention(self.q64, self.k64, self.v64, self.table, self.lengths, self.starts, self.scale, self.prefix, self.prefix_len)

    def compare(self, out, lse, weigh=False):
        want, want_lse, weights, spread = self.expected()
        T = int(self.starts[-1])
        got = out[:T].double().cpu().numpy()
        u = HALF_STEP[self.ty]
        # the result's rounding, the weights' rounding to the cache's type (of 16-bit queries), and the f32 sums
        bound = u * np.abs(want[:T]) + (u * spread[:T] if self.ty != "f32" else 0) + F32_TOL * max(np.abs(self.v64[np.isfinite(self.v64)]).max(initial=0), 1e-30)
        assert np.all(np.abs(got - want[:T]) <= bound), np.max(np.abs(got - want[:T]) / bound)
        gl = lse[:T].double().cpu().numpy()
        seen = np.isfinite(want_lse[:T])
        assert np.array_equal(seen, np.isfinite(gl)) and np.all(gl[~seen] == -np.inf)
        assert np.all(np.abs(gl[seen] - want_lse[:T][seen]) <= F32_TOL * np.maximum(1, np.abs(want_lse[:T][seen])))
        mass = self.mass.cpu().numpy()
        if weigh:
            for b in range(len(self.lengths)):
                n = self.lengths[b]
                w = self.mass0[b, :, :n].astype(np.float64) + weights[b, :, :n]
                assert np.all(np.abs(mass[b, :, :n] - w) <= F32_TOL * np.maximum(w, 1))
                assert np.array_equal(mass[b, :, n:], self.mass0[b, :, n:], equal_nan=True)
        else:
            assert np.array_equal(mass, self.mass0, equal_nan=True)
        self.c.check()


ATTENTION = [  # type, H, G, D, own lengths, tokens per sequence (None: one each), prefix, padding rows
    ("f32", 8, 2, 64, [1], None, 0, 0),
    ("f32", 8, 2, 64, [65], None, 0, 0),
    ("f32", 32, 8, 128, [1, 63, 64, 65, 700, 2], None, 0, 0),
    ("f32", 32, 8, 128, [0, 5, 0, 130], None, 0, 0),       # rows that see nothing
    ("f32", 32, 8, 128, [0, 5, 0, 130], None, 1, 0),       # the prefix alone
    ("f16", 32, 8, 128, [33, 1, 200], None, 63, 0),
    ("bf16", 32, 8, 128, [33, 1, 200], None, 64, 0),
    ("bf16", 16, 2, 64, [17] * 9, None, 65, 0),
    ("f16", 8, 8, 64, [300, 7], None, 1000, 0),            # one head per group
    ("f32", 16, 1, 128, [90, 40, 3], None, 129, 0),        # sixteen heads per group
    ("bf16", 6, 2, 128, [90, 40, 3], None, 129, 0),        # three heads per group
    ("f16", 10, 2, 64, [500, 1], None, 20, 0),             # five
    ("f16", 32, 4, 128, [1500, 4100], None, 300, 0),
    ("bf16", 32, 8, 128, [20] * 70, None, 500, 0),         # more pooled rows than one tile
    ("f32", 32, 8, 128, [10 + i for i in range(40)], None, 2100, 0),
    ("f32", 32, 8, 128, [33, 2, 1, 64], [33, 2, 1, 64], 0, 0),       # fresh prompts
    ("f32", 32, 8, 128, [70, 9, 0, 300], [30, 9, 0, 17], 100, 5),    # later chunks, a sequence without tokens, padding
    ("f16", 32, 8, 128, [70, 9, 4, 300], [30, 9, 0, 17], 100, 3),
    ("bf16", 16, 8, 128, [400, 260], [400, 130], 77, 0),
    ("bf16", 8, 2, 64, [150, 2, 70], [150, 2, 1], 200, 1),
    ("f16", 8, 1, 64, [129, 65, 1], [64, 65, 1], 0, 0),
    ("f32", 8, 2, 64, [5, 200], [9, 200], 0, 0),           # more tokens than slots: the first four see nothing
    ("f16", 6, 2, 128, [140, 33], [140, 33], 64, 0),       # three heads per group: tiles that cut tokens
    ("f32", 10, 2, 128, [140, 33], [40, 33], 10, 2),
    ("bf16", 32, 8, 128, [1000], [1000], 300, 0),
    ("f32", 8, 2, 64, [2500, 1100], [1500, 40], 50, 0),    # row tiles that see none of the last slots
    ("bf16", 12, 2, 128, [3100, 7], [1300, 7], 0, 1),
    ("f16", 8, 8, 128, [1025, 1024, 2049], [1, 300, 260], 0, 0),
]


@pytest.mark.parametrize("weigh", [False, True])
@pytest.mark.parametrize("case", range(len(ATTENTION)))
def test_attention(torch, case, weigh):
    ty, H, G, D, lengths, tokens, prefix, pad = ATTENTION[case]
    s = Case(torch, ty, H, G, D, lengths, tokens, prefix, layered=case % 2 == 1, spare=case % 3, pad=pad, seed=case)
    before = torch.full_like(s.q, 7.0)
    out, lse = s.attend(weigh=weigh, out=before)
    assert out is before
    s.compare(out, lse, weigh)
    if pad:
        assert torch.all(out[-pad:] == 7.0)


@pytest.mark.parametrize("ty", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("tokens", [None, [3, 70]])
def test_attention_large_scores(torch, ty, tokens):
    """Scores of some hundreds: one position holds nearly all the weight and the running maximum climbs."""
    s = Case(torch, ty, 8, 2, 128, [300, 200], tokens, 500, k_scale=12.0, seed=5)
    # 2^-24 of a score of ~1,000 (base 2) is off by 6e-5 in the exponent: weights and lse to that
    want, want_lse, _, spread = s.expected()
    out, lse = s.attend()
    u = HALF_STEP[ty]
    big = np.abs(want_lse).max() / math.log(2) * 2.0 ** -21
    bound = u * np.abs(want) + (u if ty != "f32" else 0) * spread + (big + F32_TOL) * 4.0
    assert np.all(np.abs(out.double().cpu().numpy() - want) <= bound)
    assert np.all(np.abs(lse.double().cpu().numpy() - want_lse) <= F32_TOL * np.abs(want_lse))


def test_attention_tiny_and_huge_queries(torch):
    """f32 rows whose elements are subnormal (all scores 0: the mean of v) or near the type's top."""
    s = Case(torch, "f32", 8, 2, 64, [40, 40], None, 0, seed=9)
    s.q[0] = 1e-42
    s.q[1] = s.q[1] * 1e30
    s.scale = 1e-30
    s.q64 = s.q.double().cpu().numpy()
    out, lse = s.attend(scale=s.scale)
    s.compare(out, lse)


def test_attention_nan_stays_in_its_row(torch):
    s = Case(torch, "f32", 8, 2, 128, [70, 30], None, 40, seed=3)
    s.q[1, 2] = float("nan")
    out, lse = s.attend()
    bad = torch.zeros(2, 8, dtype=torch.bool, device="cuda")
    bad[1, 2] = True
    assert torch.equal(torch.isnan(out).all(-1), bad) and torch.equal(torch.isnan(out).any(-1), bad)
    assert torch.equal(torch.isnan(lse), bad)


def test_attention_without_tokens(torch):
    s = Case(torch, "f16", 8, 2, 64, [3, 4], [0, 0], 0)
    out, lse = s.attend(weigh=True)
    assert out.shape == (0, 8, 64) and np.array_equal(s.mass.cpu().numpy(), s.mass0, equal_nan=True)


def test_attention_packed_queries_and_output(torch):
    """q as a slice of packed QKV rows, out as a slice of wider rows."""
    s = Case(torch, "bf16", 8, 2, 64, [50, 60], None, 70, seed=4)
    wide = torch.zeros(2, 16, 64, dtype=torch.bfloat16, device="cuda")
    wide[:, 4:12] = s.q
    to = torch.full((2, 9, 64), 3.0, dtype=torch.bfloat16, device="cuda")
    s.q = wide[:, 4:12]
    out, lse = s.attend(out=to[:, 1:])
    s.compare(out, lse)
    assert torch.all(to[:, 0] == 3.0)


@pytest.mark.parametrize("ty", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("H,G,D", [(8, 2, 64), (32, 8, 128), (6, 2, 128), (16, 1, 64)])
@pytest.mark.parametrize("tokens", [None, [1, 0, 70, 5]])
@pytest.mark.parametrize("norm", [True, False])
def test_append(torch, ty, H, G, D, tokens, norm):
    from fish_s2pro_b200 import PagedKvCache
    rng = np.random.default_rng(H + D)
    B, per = 4, 3
    kv = torch.bfloat16 if ty == "bf16" else torch.float16
    past = np.array([0, 63, 100, 64], np.int32)
    counts = [1] * B if tokens is None else tokens
    starts = np.concatenate([[0], np.cumsum(counts)])
    T, pad = int(starts[-1]), 0 if tokens is None else 3
    table = rng.permutation(B * per).reshape(B, per).astype(np.int32)
    pos = rng.integers(0, 32768, T + pad).astype(np.int32)
    pos[:3] = [0, 2 ** 31 - 1, -5]
    dt = act_dtype(torch, ty)
    (q64, q), (k64, k), (v64, v) = (rounded(torch, rng.standard_normal((T + pad, n, D)) * 1.7, dt) for n in (H, G, G))
    gains = [(1 + 0.2 * rng.standard_normal(D)).astype(np.float32) if norm else None for _ in range(2)]
    dev = lambda x: None if x is None else torch.from_numpy(np.ascontiguousarray(x)).cuda()
    kp, vp = (torch.full((B * per, G, PAGE, D), 9.0, dtype=kv, device="cuda") for _ in range(2))
    lengths = torch.full((B,), -1, dtype=torch.int32, device="cuda")
    positions = torch.full((B, G, per * PAGE), -7, dtype=torch.int32, device="cuda")
    mass = torch.full((B, G, per * PAGE), 5.0, device="cuda")
    c = PagedKvCache(kp, vp, dev(table), lengths, positions=positions, mass=mass)
    before = torch.full_like(q, 7.0)
    got = c.append(q, k, v, dev(pos), dev(past), q_start=None if tokens is None else dev(starts.astype(np.int32)), q_norm=dev(gains[0]),
                   k_norm=dev(gains[1]), eps=1e-6, rope_base=1e6, out=before)
    c.check()
    # norm: sum of squares, rsqrt (2 ulp), two products; rotation: angle pi 2^-25 off, sines 2 ulp, two products and a sum: under
    # 2^-20 of the pair's size in all
    def close(got, want, u):
        pair = np.repeat(np.sqrt(want[..., 0::2] ** 2 + want[..., 1::2] ** 2), 2, -1)
        assert np.all(np.abs(got - want) <= 2.0 ** -20 * pair + u * np.abs(want) + 1e-30)
    want_q, want_k = ref.rotate(q64[:T], gains[0], pos[:T], 1e-6, 1e6), ref.rotate(k64[:T], gains[1], pos[:T], 1e-6, 1e6)
    close(got[:T].double().cpu().numpy(), want_q, HALF_STEP[ty])
    assert torch.all(got[T:] == 7.0)
    k_all, v_all = kp.double().cpu().numpy(), vp.double().cpu().numpy()
    touched = np.zeros((B * per, PAGE), bool)
    for b in range(B):
        for i in range(counts[b]):
            t, slot = int(starts[b]) + i, int(past[b]) + i
            page, r = table[b, slot // PAGE], slot % PAGE
            touched[page, r] = True
            close(k_all[page, :, r], want_k[t], HALF_STEP["bf16" if ty == "bf16" else "f16"] + 2.0 ** -24)
            assert np.array_equal(v_all[page, :, r], torch.from_numpy(v64[t]).to(kv).double().numpy())
            assert torch.all(positions[b, :, slot] == int(pos[t])) and torch.all(mass[b, :, slot] == 0)
        free = np.ones(per * PAGE, bool)
        free[past[b]: past[b] + counts[b]] = False
        assert torch.all(positions[b][:, dev(free)] == -7) and torch.all(mass[b][:, dev(free)] == 5.0)
    assert np.all(k_all.transpose(0, 2, 1, 3)[~touched] == 9.0) and np.all(v_all.transpose(0, 2, 1, 3)[~touched] == 9.0)
    assert lengths.tolist() == [int(p) + n for p, n in zip(past, counts)]


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("counts", [[593], [700, 0, 1, 1200, 0, 333], [0, 9000, 1, 0, 31, 10100, 7]])
def test_append_of_many_tokens(torch, counts, D):
    """More tokens than blocks that run at once: groups of tokens that cross sequences, pages and empty sequences."""
    from fish_s2pro_b200 import PagedKvCache
    rng = np.random.default_rng(sum(counts))
    B, H, G, T = len(counts), 2, 1, sum(counts)
    past = rng.integers(0, 70, B).astype(np.int32)
    per = -(-int((past + counts).max()) // PAGE)
    starts = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    table = rng.permutation(B * per).reshape(B, per).astype(np.int32)
    pos = rng.integers(0, 100000, T).astype(np.int32)
    (q64, q), (k64, k), (v64, v) = (rounded(torch, rng.standard_normal((T, n, D)), torch.float32) for n in (H, G, G))
    gain = (1 + 0.2 * rng.standard_normal(D)).astype(np.float32)
    dev = lambda x: torch.from_numpy(np.ascontiguousarray(x)).cuda()
    kp, vp = (torch.full((B * per, G, PAGE, D), 9.0, dtype=torch.float16, device="cuda") for _ in range(2))
    positions = torch.full((B, G, per * PAGE), -7, dtype=torch.int32, device="cuda")
    c = PagedKvCache(kp, vp, dev(table), dev(np.zeros(B, np.int32)), positions=positions)
    got = c.append(q, k, v, dev(pos), dev(past), q_start=dev(starts), q_norm=dev(gain), eps=1e-6, rope_base=1e6)
    c.check()
    seq = np.repeat(np.arange(B), counts)
    slot = past[seq] + np.arange(T) - starts[seq]
    page, r = table[seq, slot // PAGE], slot % PAGE
    for have, want, u in ((got, ref.rotate(q64, gain, pos, 1e-6, 1e6), HALF_STEP["f32"]),
                          (kp[dev(page).long(), :, dev(r).long()], ref.rotate(k64, None, pos, 1e-6, 1e6), HALF_STEP["f16"] + 2.0 ** -24)):
        pair = np.repeat(np.sqrt(want[..., 0::2] ** 2 + want[..., 1::2] ** 2), 2, -1)
        assert np.all(np.abs(have.double().cpu().numpy() - want) <= 2.0 ** -20 * pair + u * np.abs(want) + 2.0 ** -25)  # f16's smallest half step
    assert torch.equal(vp[dev(page).long(), :, dev(r).long()], v.half())
    want = np.full((B, per * PAGE), -7, np.int32)
    want[seq, slot] = pos
    assert np.array_equal(positions[:, 0].cpu().numpy(), want)
    free = np.ones((B * per, PAGE), bool)
    free[page, r] = False
    assert torch.all(kp[:, 0][dev(free)] == 9.0) and torch.all(vp[:, 0][dev(free)] == 9.0)
    assert c.lengths.tolist() == (past + counts).tolist()


def test_append_in_place_from_packed_rows(torch):
    """q, k and v as slices of packed QKV rows, the queries rotated in place; no positions or mass."""
    from fish_s2pro_b200 import PagedKvCache
    rng = np.random.default_rng(1)
    packed64, packed = rounded(torch, rng.standard_normal((2, 12, 64)), torch.float32)
    kp, vp = (torch.zeros(2, 2, PAGE, 64, dtype=torch.float16, device="cuda") for _ in range(2))
    ints = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")
    c = PagedKvCache(kp, vp, ints(1, 0).view(2, 1), ints(0, 0))
    q = packed[:, :8]
    got = c.append(q, packed[:, 8:10], packed[:, 10:], ints(70, 900), ints(4, 9), out=q)
    assert got.data_ptr() == packed.data_ptr()
    want = ref.rotate(packed64[:, :10], None, np.array([70, 900]), 1e-6, 1e6)
    assert np.max(np.abs(packed[:, :8].double().cpu().numpy() - want[:, :8])) < 2.0 ** -20 * 4
    assert np.max(np.abs(kp[1, :, 4].double().cpu().numpy() - want[0, 8:])) < 2.0 ** -9
    assert torch.equal(vp[0, :, 9], packed[1, 10:].half())
    assert torch.equal(packed[:, 8:].double().cpu(), torch.from_numpy(packed64[:, 8:]))
    assert c.lengths.tolist() == [5, 10]


def evict_case(torch, lengths, budget, recent, G=3, D=64, kv="f16", seed=0, edit=None, layered=False, spare=0):
    from fish_s2pro_b200 import PagedKvCache
    rng = np.random.default_rng(seed)
    dt = torch.float16 if kv == "f16" else torch.bfloat16
    B, per = len(lengths), max(1, -(-max(lengths) // PAGE)) + spare
    table = rng.permutation(B * per + 2)[: B * per].reshape(B, per).astype(np.int32)
    pool = torch.randn(B * per + 2, 2, G, PAGE, D, generator=torch.Generator().manual_seed(seed)).to(dt)
    slots = per * PAGE
    mass = (rng.random((B, G, slots)) ** 4).astype(np.float32)
    mass[rng.random(mass.shape) < 0.3] = 0.0  # ties
    pos = np.stack([[rng.permutation(slots) for _ in range(G)] for _ in range(B)]).astype(np.int32)
    if edit:
        edit(mass, pos, rng)
    dev = lambda x: torch.from_numpy(np.ascontiguousarray(x)).cuda()
    dpool = pool.cuda()
    k, v = (dpool[:, 0], dpool[:, 1]) if layered else (dpool[:, 0].contiguous(), dpool[:, 1].contiguous())
    dmass, dpos, past = dev(mass), dev(pos), torch.full((B,), -1, dtype=torch.int32, device="cuda")
    c = PagedKvCache(k, v, dev(table), dev(np.asarray(lengths, np.int32)), positions=dpos, mass=dmass)
    c.evict(budget, recent, past)
    c.check()
    want = pool.view(torch.int16).numpy().copy()
    wm, wp = mass.copy(), pos.copy()
    for b in range(B):
        for g in range(G):
            to, fro = ref.evict(pos[b, g], mass[b, g], lengths[b], budget, recent)
            for i, j in zip(to, fro):
                want[table[b, i // PAGE], :, g, i % PAGE] = want[table[b, j // PAGE], :, g, j % PAGE]
                wm[b, g, i], wp[b, g, i] = wm[b, g, j], wp[b, g, j]
    assert past.tolist() == [min(n, budget) for n in lengths]
    assert c.lengths.tolist() == list(lengths)
    assert np.array_equal(dpos.cpu().numpy(), wp)
    assert np.array_equal(dmass.cpu().numpy().view(np.int32), wm.view(np.int32))
    assert np.array_equal(k.contiguous().cpu().view(torch.int16).numpy(), want[:, 0])
    assert np.array_equal(v.contiguous().cpu().view(torch.int16).numpy(), want[:, 1])


def _odd_mass(mass, pos, rng):
    flat = mass.reshape(-1)
    for x in (np.nan, np.inf, -np.inf, -0.0, 1e-42, -1.0):
        flat[rng.integers(0, flat.size, 40)] = x


def _equal_mass(mass, pos, rng):
    mass[:] = 0.25


def _same_positions(mass, pos, rng):
    pos[:] = 11


EVICT = [  # lengths, budget, recent, keywords
    ([1, 2, 0], 1, 0, {}),
    ([1, 2, 5], 1, 1, {}),
    ([64, 65, 63, 200], 64, 10, {}),
    ([65], 64, 64, {}),
    ([700, 1300, 130], 128, 32, dict(kv="bf16", D=128)),
    ([1500, 2049], 1000, 500, dict(layered=True)),
    ([2049] * 3, 2048, 512, dict(spare=1)),
    ([5000], 17, 3, {}),
    ([5000], 4990, 0, {}),
    ([400, 900], 300, 50, dict(edit=_odd_mass)),
    ([400, 900], 300, 0, dict(edit=_equal_mass)),
    ([400, 900], 300, 7, dict(edit=_same_positions)),   # every slot is recent: the lowest stay
    ([130, 700], 5000, 100, {}),                        # within the budget: untouched
    ([9000], 4096, 1024, dict(G=2)),
    ([33000, 20], 16384, 100, dict(G=1)),
]


@pytest.mark.parametrize("case", range(len(EVICT)))
def test_evict(torch, case):
    lengths, budget, recent, kw = EVICT[case]
    evict_case(torch, lengths, budget, recent, seed=case, **kw)


def test_decode_loop_keeps_its_budget(torch):
    """append -> attention with weights -> evict over one shared prefix, step by step against the plain forms: sequences of
    different lengths grow to the budget and stay there.  The choice of what to evict is checked on the device's own mass (the
    reference's differs in the last bits), everything else on the reference's values."""
    s = Case(torch, "f32", 8, 2, 64, [5, 37, 40], None, 70, spare=1, seed=21)
    B, G, D, budget, recent = 3, 2, 64, 40, 8
    rng = np.random.default_rng(2)
    past = s.ints(s.lengths)
    seen = s.lengths.astype(np.int64).copy()
    k64, v64, pos_ref = s.k64.copy(), s.v64.copy(), s.pos0.copy()
    for step in range(12):
        pos = 70 + seen
        (q64, q), (kn64, kn), (vn64, vn) = (rounded(torch, rng.standard_normal((B, n, D)), torch.float32) for n in (8, G, G))
        have = past.cpu().numpy()
        qr = s.c.append(q, kn, vn, s.ints(pos), past)
        lengths = have + 1
        assert s.c.lengths.tolist() == lengths.tolist()
        kr = ref.rotate(kn64, None, pos, 0.0, 1e6)
        for b in range(B):
            page, r = s.table[b, have[b] // PAGE], have[b] % PAGE
            k64[page, :, r], v64[page, :, r] = torch.from_numpy(kr[b]).half().double().numpy(), torch.from_numpy(vn64[b]).half().double().numpy()
            pos_ref[b, :, have[b]] = pos[b]
        mass = s.mass.cpu().numpy()
        out, lse = s.c.attention(qr, prefix_pages=s.prefix_pages, prefix_len=70, weigh=True, return_lse=True)
        want, want_lse, weights, _ = ref.attention(ref.rotate(q64, None, pos, 0.0, 1e6), k64, v64, s.table, lengths, np.arange(B + 1),
                                                   s.scale, s.prefix, 70)
        # keys may differ from the reference's by an f16 step where the rotation rounds the other way: 2^-10 of a key in one score
        assert np.max(np.abs(out.double().cpu().numpy() - want)) < 2e-3
        after = s.mass.cpu().numpy()
        for b in range(B):
            n = lengths[b]
            assert np.max(np.abs(after[b, :, :n] - mass[b, :, :n] - weights[b, :, :n])) < 2e-3
        s.c.evict(budget, recent, past)
        for b in range(B):
            for g in range(G):
                to, fro = ref.evict(pos_ref[b, g], after[b, g], lengths[b], budget, recent)
                for i, j in zip(to, fro):
                    for x in (k64, v64):
                        x[s.table[b, i // PAGE], g, i % PAGE] = x[s.table[b, j // PAGE], g, j % PAGE]
                    pos_ref[b, g, i] = pos_ref[b, g, j]
        assert past.tolist() == [min(n, budget) for n in lengths]
        got_pos = s.positions.cpu().numpy()
        for b in range(B):
            n = min(lengths[b], budget)
            assert np.array_equal(got_pos[b, :, :n], pos_ref[b, :, :n])
        seen += 1
    s.c.check()


# ---------------------------------------------------------------------------
# how the calls are used: streams, graphs, long pools, many sequences, bad tables
# ---------------------------------------------------------------------------


def test_attention_on_another_stream(torch):
    """Enqueued on torch's current stream, behind that stream's work, whatever ran on the default one."""
    s = Case(torch, "f32", 8, 2, 128, [200, 90], None, 300, seed=31)
    side = torch.cuda.Stream()
    q, zero = s.q.clone(), torch.zeros_like(s.q)
    s.q = zero
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)
        zero.copy_(q)
        out, lse = s.attend()
    side.synchronize()
    s.compare(out, lse)


@pytest.mark.parametrize("ty,tokens", [("f32", None), ("bf16", None), ("bf16", [40, 7, 130])])
def test_attention_in_graphs_that_run_together(torch, ty, tokens):
    """Two captured calls over different queries, replayed at the same time on two streams, many times: each has a workspace of
    its own, and every replay gives what the eager call gave, bit for bit."""
    s = Case(torch, ty, 32, 8, 128, [300, 700, 130], tokens, 900, seed=32)
    qs = [s.q.clone(), s.q.flip(0).contiguous()]
    eager = []
    for q in qs:
        s.q = q
        eager.append([x.clone() for x in s.attend()])
    graphs, outs = [], []
    for q in qs:
        s.q = q
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(s.attend())
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in graphs]
    torch.cuda.synchronize()
    for _ in range(20):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for (out, lse), (want, want_lse) in zip(outs, eager):
        assert torch.equal(out, want) and torch.equal(lse, want_lse)
    s.c.check()


def test_decode_step_in_a_graph(torch):
    """append, attention with weights, evict and the position counter captured once; replays carry the lengths on, on the device.
    The same steps run eagerly on a copy give the same bits."""
    from fish_s2pro_b200 import PagedKvCache
    a = Case(torch, "f16", 8, 2, 64, [10, 30, 33], None, 100, spare=1, seed=33)
    states = []
    for _ in range(2):
        k, v, mass, pos = (x.clone() for x in (a.c.k, a.c.v, a.mass, a.positions))
        mass.nan_to_num_(0.0)
        c = PagedKvCache(k, v, a.c.page_table, a.ints(a.lengths), positions=pos, mass=mass)
        states.append(dict(c=c, past=a.ints(a.lengths), pos=a.ints(100 + a.lengths), q=a.q.clone()))
    gen = torch.Generator(device="cuda").manual_seed(1)
    new = [torch.randn(3, 2, 64, dtype=torch.float16, device="cuda", generator=gen) for _ in range(2)]

    def step(s):
        q = s["c"].append(s["q"], new[0], new[1], s["pos"], s["past"])
        out = s["c"].attention(q, prefix_pages=a.prefix_pages, prefix_len=100, weigh=True)
        s["c"].evict(32, 4, s["past"])
        s["pos"].add_(1)
        return out

    eager = [step(states[0]).clone() for _ in range(9)]
    g = torch.cuda.CUDAGraph()
    kept = {x: states[1][x].clone() for x in ("past", "pos")}
    with torch.cuda.graph(g):
        out = step(states[1])
    for x, v in kept.items():
        assert torch.equal(states[1][x], v)  # capturing ran nothing
    for want in eager:
        g.replay()
        assert torch.equal(out, want)
    for x in ("k", "v", "mass", "positions", "lengths"):
        u, w = (getattr(s["c"], x) for s in states)
        assert torch.equal(u.nan_to_num(0.0) if u.is_floating_point() else u, w.nan_to_num(0.0) if w.is_floating_point() else w)
    assert torch.equal(states[0]["past"], states[1]["past"]) and states[0]["past"].tolist() == [19, 32, 32]


@pytest.mark.parametrize("tokens", [None, [9, 140]])
def test_pool_past_2_to_the_32_elements(torch, tokens):
    """Pages whose rows lie more than 2^32 elements into the pool: append, attention with weights and eviction there."""
    from fish_s2pro_b200 import PagedKvCache
    s = Case(torch, "f16", 8, 2, 128, [70, 300], tokens, 130, seed=34)
    n = s.c.n_pages
    per_page = 2 * PAGE * 128
    far = 2 ** 32 // per_page + 1000
    k, v = (torch.empty(far + n, 2, PAGE, 128, dtype=torch.float16, device="cuda") for _ in range(2))
    k[far:], v[far:] = s.c.k, s.c.v
    c = PagedKvCache(k, v, s.c.page_table + far, s.c.lengths, positions=s.positions, mass=s.mass)
    s.c = c
    s.prefix_pages = s.prefix_pages + far
    out, lse = s.attend(weigh=True)
    s.compare(out, lse, weigh=True)
    before = [x[far:].clone() for x in (k, v)]
    mass0, pos0 = s.mass.cpu().numpy(), s.positions.cpu().numpy()
    c.evict(64, 8, s.ints([0, 0]))
    c.check()
    for b, n_b in enumerate(s.lengths):
        for g in range(2):
            to, fro = ref.evict(pos0[b, g], mass0[b, g], int(n_b), 64, 8)
            for i, j in zip(to, fro):
                for x in before:
                    x[s.table[b, i // PAGE], g, i % PAGE] = x[s.table[b, j // PAGE], g, j % PAGE]
    assert all(torch.equal(x[far:].view(torch.int16), y.view(torch.int16)) for x, y in zip((k, v), before))
    q = torch.randn(2, 8, 128, dtype=torch.float16, device="cuda")
    kn = torch.randn(2, 2, 128, dtype=torch.float16, device="cuda")
    c.append(q, kn, kn, s.ints([1, 2]), s.ints([5, 60]), eps=0.0)
    c.check()
    assert torch.equal(v[far + int(s.table[0, 0]), :, 5], kn[0]) and torch.equal(v[far + int(s.table[1, 0]), :, 60], kn[1])


def test_many_sequences(torch):
    """A thousand short sequences, some empty, some without a token of theirs; the same page under two of them."""
    rng = np.random.default_rng(35)
    lengths = rng.integers(0, 90, 1000)
    tokens = np.minimum(lengths, rng.integers(0, 4, 1000)).astype(int)
    s = Case(torch, "bf16", 6, 2, 64, lengths.tolist(), tokens.tolist(), 80, seed=35, pad=2)
    s.table[17] = s.table[500]  # sequence 17 reads 500's pages
    n = int(min(lengths[17], lengths[500]))
    s.lengths[17] = n
    if tokens[17] > n:
        tokens[17] = n
    s.c.page_table[17] = s.c.page_table[500]
    s.c.lengths[17] = n
    s.mass0[17] = 0.5
    s.mass[17] = 0.5
    out, lse = s.attend(weigh=True)
    s.compare(out, lse, weigh=True)


@pytest.mark.parametrize("ty,n_seq,longest,prefix", [("bf16", 40, 5, 700), ("f32", 40, 70, 100), ("f32", 70, 40, 700), ("f16", 70, 100, 130), ("bf16", 64, 2, 9000)])
def test_ragged_batches_behind_a_prefix(torch, ty, n_seq, longest, prefix):
    """More row tiles than SMs, few rows or many behind short and long prefixes, up to 64 sequences and more."""
    rng = np.random.default_rng(36)
    tokens = rng.integers(0, longest + 1, n_seq)
    tokens[3] = 0
    lengths = tokens + rng.integers(0, 200, n_seq) * rng.integers(0, 2, n_seq)
    s = Case(torch, ty, 16, 8, 64, lengths.tolist(), tokens.tolist(), prefix, seed=36, pad=1)
    out, lse = s.attend(weigh=True)
    s.compare(out, lse, weigh=True)


@pytest.mark.parametrize("ty,D", [("bf16", 128), ("f32", 128), ("f16", 64)])
def test_short_sequences_beside_long_ones(torch, ty, D):
    """Positions are split by the longest sequence's slots, so most of the short ones' ranges are empty: many calls, as these
    items need no products and their threads run ahead."""
    s = Case(torch, ty, 12, 2, D, [3100, 7, 1, 0, 130, 64], [300, 7, 1, 0, 30, 2], 0, seed=37)
    first = [x.clone() for x in s.attend()]
    s.compare(*first)
    for _ in range(100):
        assert all(torch.equal(x, y) for x, y in zip(first, s.attend()))
    s.c.check()


def test_results_do_not_change_from_call_to_call(torch):
    """Weights and outputs are summed in a fixed order: repeated calls give the same bits."""
    for tokens in (None, [300, 20, 77]):
        s = Case(torch, "f32", 16, 4, 128, [900, 20, 400], tokens, 1500, seed=36)
        first = None
        for _ in range(5):
            s.mass.zero_()
            out, lse = s.attend(weigh=True)
            got = [out.clone(), lse.clone(), s.mass.clone()]
            first = first or got
            assert all(torch.equal(x, y) for x, y in zip(first, got))


@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("page", [-1, "n_pages", 2 ** 31 - 1, -2 ** 31])
def test_bad_pages_are_reported_and_stay_in_their_sequence(torch, page, ragged):
    from fish_s2pro_b200 import S2dError
    s = Case(torch, "f16", 8, 2, 128, [130, 150, 70], [3, 60, 2] if ragged else None, 100, seed=37)
    want, *_ = s.expected()
    s.c.page_table[1, 1] = s.c.n_pages if page == "n_pages" else page
    mass0 = s.mass.clone()
    out, lse = s.attend(weigh=True)
    with pytest.raises(S2dError, match="page id outside the pool"):
        s.c.check()
    s.c.check()  # cleared
    rows = np.r_[: s.starts[1], s.starts[2]: s.starts[3]]
    assert np.max(np.abs(out.double().cpu().numpy()[rows] - want[rows])) < 1e-2
    assert torch.all(s.mass[[0, 2]].nan_to_num(0) >= mass0[[0, 2]].nan_to_num(0))
    before = s.c.k.clone().view(torch.int16)
    s.positions.copy_(torch.from_numpy(s.pos0))
    s.mass.copy_(torch.from_numpy(s.mass0))
    s.c.evict(100, 10, s.ints([0, 0, 0]))
    with pytest.raises(S2dError, match="page id outside the pool"):
        s.c.check()
    untouched = np.setdiff1d(np.arange(s.c.n_pages), s.table[:2].reshape(-1))
    assert torch.equal(s.c.k.view(torch.int16)[untouched], before[untouched])
    q = torch.zeros(3, 8, 128, dtype=torch.float16, device="cuda")
    kn = torch.ones(3, 2, 128, dtype=torch.float16, device="cuda")
    before = s.c.v.clone().view(torch.int16)
    s.c.append(q, kn, kn, s.ints([1, 2, 3]), s.ints([130, 64, 70]))
    with pytest.raises(S2dError, match="page id outside the pool"):
        s.c.check()
    changed = (s.c.v.view(torch.int16) != before).any(-1).any(-1).any(-1).nonzero().flatten().tolist()
    assert sorted(changed) == sorted(int(s.table[b, n // PAGE]) for b, n in ((0, 130), (2, 70)))


@pytest.mark.parametrize("length", [-1, 2 ** 31 - 1, -2 ** 31, 193])
@pytest.mark.parametrize("ragged", [False, True])
def test_bad_lengths_are_reported(torch, length, ragged):
    """Lengths outside the page table (three pages here): held inside it."""
    from fish_s2pro_b200 import S2dError
    s = Case(torch, "f16", 8, 2, 128, [130, 150, 70], [3, 60, 2] if ragged else None, 100, seed=38)
    want, *_ = s.expected()
    s.c.lengths[1] = length
    out, lse = s.attend(weigh=True)
    with pytest.raises(S2dError, match="out of range"):
        s.c.check()
    rows = np.r_[: s.starts[1], s.starts[2]: s.starts[3]]
    assert np.max(np.abs(out.double().cpu().numpy()[rows] - want[rows])) < 1e-2
    s.c.evict(100, 10, s.ints([0, 0, 0]))
    with pytest.raises(S2dError, match="out of range"):
        s.c.check()


@pytest.mark.parametrize("starts", [[0, 40, 20, 60], [0, -3, 20, 60], [0, 20, 100, 60], [-5, 20, 40, 60], [7, 20, 40, 60], [0, 20, 40, 1000], [0, 0, 0, -1]])
def test_bad_starts_touch_nothing_else(torch, starts):
    """q_start out of order or out of range: reported where it is (a first entry above 0 just leaves rows out), no row past the
    tokens written."""
    from fish_s2pro_b200 import S2dError
    s = Case(torch, "bf16", 8, 2, 64, [130, 150, 70], [20, 20, 20], 100, seed=39)
    s.q_start = s.ints(starts)
    wide = torch.full((70, 8, 64), 5.0, dtype=torch.bfloat16, device="cuda")
    s.attend(weigh=True, out=wide[:60])
    assert torch.all(wide[60:] == 5.0)
    if starts != [7, 20, 40, 60]:
        with pytest.raises(S2dError, match="out of range"):
            s.c.check()
    kn = torch.zeros(60, 2, 64, dtype=torch.bfloat16, device="cuda")
    s.c.append(s.q, kn, kn, s.ints(range(60)), s.ints([130, 150, 70]), q_start=s.q_start, out=wide[:60])
    assert torch.all(wide[60:] == 5.0)
    with pytest.raises(S2dError):
        s.c.check()


def test_append_to_a_full_sequence_and_bad_past(torch):
    from fish_s2pro_b200 import S2dError
    for past, message in ((190, "past the last slot"), (192, "past the last slot"), (193, "out of range"), (-1, "out of range"), (2 ** 31 - 1, "out of range")):
        s = Case(torch, "f16", 8, 2, 64, [64, 192, 64], [2, 5, 2], 0, seed=40)
        kn = torch.ones(9, 2, 64, dtype=torch.float16, device="cuda")
        before = s.c.v.clone()
        s.c.append(s.q, kn, kn, s.ints(range(9)), s.ints([10, past, 20]), q_start=s.q_start)
        with pytest.raises(S2dError, match=message):
            s.c.check()
        assert s.c.lengths.tolist() == [12, min(192, max(past, 0) + 5) if past < 2 ** 31 - 1 else 192, 22]
        after = s.c.v
        assert torch.all(after[int(s.table[0, 0]), :, 10:12] == 1) and torch.all(after[int(s.table[2, 0]), :, 20:22] == 1)
        tail = after[int(s.table[1, 2])]
        if past == 190:
            assert torch.all(tail[:, 62:] == 1)
            tail = tail[:, :62]
            assert torch.equal(tail, before[int(s.table[1, 2])][:, :62])
        else:
            assert all(torch.equal(after[int(p)], before[int(p)]) for p in s.table[1])


def test_refusals(torch):
    from fish_s2pro_b200 import PagedKvCache, S2dError
    s = Case(torch, "f16", 8, 2, 64, [30, 40], None, 70, seed=41)
    c, q = s.c, s.q
    kn = torch.zeros(2, 2, 64, dtype=torch.float16, device="cuda")
    pos, past = s.ints([1, 2]), s.ints([1, 2])
    pool = torch.zeros(4, 2, PAGE, 64, dtype=torch.float16, device="cuda")
    table, lengths = s.ints([[0, 1], [2, 3]]), s.ints([1, 1])
    calls = [
        lambda: PagedKvCache(pool.float(), pool.float(), table, lengths),
        lambda: PagedKvCache(pool, pool[:, :1], table, lengths),
        lambda: PagedKvCache(pool.transpose(1, 2), pool.transpose(1, 2), table, lengths),
        lambda: PagedKvCache(pool.cpu(), pool.cpu(), table, lengths),
        lambda: PagedKvCache(pool, pool, table.long(), lengths),
        lambda: PagedKvCache(pool, pool, table, lengths[:1]),
        lambda: PagedKvCache(pool, pool, table, lengths, mass=torch.zeros(2, 2, 64, device="cuda")),
        lambda: c.attention(q.float().double()),
        lambda: c.attention(q.bfloat16()),
        lambda: c.attention(q[:, :7]),
        lambda: c.attention(q.cpu()),
        lambda: c.attention(q.transpose(0, 1)),
        lambda: c.attention(torch.cat([q, q])),                      # four tokens, two sequences, no q_start
        lambda: c.attention(q, q_start=s.ints([0, 1])),
        lambda: c.attention(q, q_start=torch.tensor([0, 1, 2], device="cuda")),
        lambda: c.attention(q, prefix_pages=s.prefix_pages, prefix_len=129),
        lambda: c.attention(q, prefix_len=3),
        lambda: c.attention(q, prefix_pages=s.prefix_pages, prefix_len=-1),
        lambda: c.attention(q, scale=float("nan")),
        lambda: c.attention(q, scale=1e300),
        lambda: c.append(q, kn, kn, pos, past, eps=1e300),
        lambda: c.evict(2 ** 31, 5),
        lambda: c.evict(10.5, 5),
        lambda: c.attention(q, out=q[:, :4]),
        lambda: c.attention(q, out=q),
        lambda: c.attention(q.detach().clone().requires_grad_()),
        lambda: c.attention(q, out=torch.empty(2 * 8 * 64 + 1, dtype=torch.float16, device="cuda")[1:].view(2, 8, 64)),  # misaligned
        lambda: c.append(q, kn, kn.float(), pos, past),
        lambda: c.append(q, kn[:1], kn, pos, past),
        lambda: c.append(q, kn, kn, pos.long(), past),
        lambda: c.append(q, kn, kn, pos, c.lengths),
        lambda: c.append(q, kn, kn, pos, past, q_norm=torch.ones(32, device="cuda")),
        lambda: c.append(q, kn, kn, pos, past, rope_base=0.0),
        lambda: c.append(q, kn, kn, pos, past, eps=-1.0),
        lambda: c.evict(0, 0),
        lambda: c.evict(10, 11),
        lambda: c.evict(10, -1),
        lambda: c.evict(10, 1, c.lengths),
        lambda: PagedKvCache(pool, pool, table, lengths).evict(1, 0),
        lambda: PagedKvCache(pool, pool, table, lengths).attention(q, weigh=True),
    ]
    for i, call in enumerate(calls):
        with pytest.raises(S2dError) as e:
            call()
        assert e.value.code == -1, i
    c.check()


def test_append_refuses_lengths_among_its_inputs(torch):
    """After past.copy_(lengths) the lengths have the values of pos, but the call writes them."""
    from fish_s2pro_b200 import S2dError
    s = Case(torch, "f16", 8, 2, 64, [30, 40], None, 0, seed=42, spare=1)
    kn = torch.zeros(2, 2, 64, dtype=torch.float16, device="cuda")
    past = s.c.lengths.clone()
    ends = torch.zeros(3, dtype=torch.int32, device="cuda")
    ends[1:] = s.c.lengths
    from fish_s2pro_b200 import PagedKvCache
    other = PagedKvCache(s.c.k, s.c.v, s.c.page_table, ends[1:])
    for call in (lambda: s.c.append(s.q, kn, kn, s.c.lengths, past), lambda: other.append(s.q, kn, kn, s.ints([1, 2]), past, q_start=ends)):
        with pytest.raises(S2dError, match="lengths") as e:
            call()
        assert e.value.code == -1
    s.c.append(s.q, kn, kn, past, past)  # pos and past may be one tensor
    s.c.check()
    assert s.c.lengths.tolist() == [31, 41]


def test_append_refuses_an_output_over_keys_or_values(torch):
    """As many query heads as KV heads: out = k has the right shape, and queries would be written over keys still to be read.
    Slices of one packed tensor lie between each other's rows and are taken."""
    from fish_s2pro_b200 import PagedKvCache, S2dError
    s = Case(torch, "f16", 2, 2, 64, [30, 40], None, 0, seed=43)
    packed = torch.randn(2, 8, 64, dtype=torch.float16, device="cuda")
    q, k, v, spare = (packed[:, i:i + 2] for i in (0, 2, 4, 6))
    past = s.ints([3, 4])
    for out in (k, v, packed[:, 1:3], packed[:, 5:7]):
        with pytest.raises(S2dError, match="q_out") as e:
            s.c.append(q, k, v, s.ints([1, 2]), past, out=out)
        assert e.value.code == -1
    before = packed.clone()
    want = s.c.append(q, k, v, s.ints([1, 2]), past)
    assert s.c.append(q, k, v, s.ints([1, 2]), past, out=spare).data_ptr() == spare.data_ptr()
    s.c.check()
    assert torch.equal(spare, want) and torch.equal(packed[:, :6], before[:, :6])


@pytest.mark.parametrize("tokens", [None, [30, 4]])
def test_attention_output_beside_the_queries(torch, tokens):
    """q and out as slices of one packed tensor, each token's output behind its queries."""
    s = Case(torch, "bf16", 8, 2, 64, [50, 60], tokens, 70, seed=44)
    packed = torch.zeros(s.q.shape[0], 17, 64, dtype=torch.bfloat16, device="cuda")
    packed[:, :8] = s.q
    s.q = packed[:, :8]
    out, lse = s.attend(out=packed[:, 9:])
    s.compare(out, lse)
    assert torch.all(packed[:, 8] == 0) and np.array_equal(packed[:, :8].double().cpu().numpy(), s.q64)


def one_above_many(torch, ty, n, gap, n_seq, G=8, tokens=None):
    """One slot (key 1, value 0) and n - 1 slots (key 0, value 1), which get 2^-gap of its weight each.  n_seq sequences over the
    same pages, or a prompt of `tokens` behind them as its prefix: (results, what all of them should be)."""
    from fish_s2pro_b200 import PagedKvCache
    D, dtype = 64, act_dtype(torch, ty)
    kv = torch.bfloat16 if ty == "bf16" else torch.float16
    k, v = torch.zeros(9, G, PAGE, D, dtype=kv, device="cuda"), torch.ones(9, G, PAGE, D, dtype=kv, device="cuda")
    k[0, :, 0, 0], v[0, :, 0] = 1.0, 0.0
    ids = torch.arange(n // PAGE, device="cuda") % 8 + 1  # the eight other pages again and again
    ids[0] = 0
    ids = ids.to(torch.int32)
    q = torch.zeros(tokens or n_seq, G, D, dtype=dtype, device="cuda")
    q[:, :, 0] = 1.0
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    if tokens:
        c = PagedKvCache(k, v, ints([[1]]), ints([0]))
        got = c.attention(q, q_start=ints([0, tokens]), prefix_pages=ids, prefix_len=n, scale=gap * math.log(2))
    else:
        c = PagedKvCache(k, v, ids.expand(n_seq, -1).contiguous(), ints([n] * n_seq))
        got = c.attention(q, scale=gap * math.log(2))
    c.check()
    w = (n - 1) * 2.0 ** -gap
    return got.double().cpu().numpy(), w / (1 + w)


@pytest.mark.parametrize("ty", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n", [8192, 32768])
@pytest.mark.parametrize("gap", [15.5, 25.05, 31.1])
def test_single_tokens_count_small_weights(torch, ty, n, gap):
    """Weights far below the largest count in the sum and in the values alike, down to where all of them together are below the
    tolerance (values are at most 1).  Enough sequences that one CTA takes each one's slots."""
    got, want = one_above_many(torch, ty, n, gap, 80)
    assert np.max(np.abs(got - want)) <= F32_TOL + (HALF_STEP[ty] * want if ty != "f32" else 0)


def periodic(torch, ty, H, G, D, n, n_seq=None, tokens=None, packed=False):
    """n positions (a multiple of 4,096) over the same 64 pages again and again, values in [1/2, 3/2]: as the prefix of `tokens`
    packed tokens, or as the slots of n_seq single ones (packed: the same by q_start).  (out, lse, what they should be): softmax
    over the period, its sum times the periods."""
    from fish_s2pro_b200 import PagedKvCache
    gen = torch.Generator(device="cuda").manual_seed(n + D)
    kv = torch.bfloat16 if ty == "bf16" else torch.float16
    k = torch.randn(64, G, PAGE, D, generator=gen, device="cuda").to(kv)
    v = (torch.rand(64, G, PAGE, D, generator=gen, device="cuda") + 0.5).to(kv)
    ids = (torch.arange(n // PAGE, device="cuda") % 64).to(torch.int32)
    q = torch.randn(tokens or n_seq, H, D, generator=gen, device="cuda").to(act_dtype(torch, ty))
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    if tokens:
        c = PagedKvCache(k, v, ints([[0]]), ints([0]))
        out, lse = c.attention(q, q_start=ints([0, tokens]), prefix_pages=ids, prefix_len=n, return_lse=True)
    else:
        c = PagedKvCache(k, v, ids.expand(n_seq, -1).contiguous(), ints([n] * n_seq))
        out, lse = c.attention(q, q_start=ints(list(range(n_seq + 1))) if packed else None, return_lse=True)
    c.check()
    rows = lambda x: x.permute(1, 0, 2, 3).reshape(G, -1, D).double()
    s = torch.einsum("tgrd,gnd->tgrn", q.double().view(-1, G, H // G, D), rows(k)) / math.sqrt(D)
    want = torch.einsum("tgrn,gnd->tgrd", s.softmax(-1), rows(v)).reshape(out.shape)
    return out.double(), lse.double(), want, torch.logsumexp(s, -1).reshape(lse.shape) + math.log(n // 4096)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("ty,n", [("f32", 8192), ("f32", 65536), ("f16", 131072), ("bf16", 524288)])
def test_single_tokens_over_long_caches(torch, ty, n, D):
    """Sums over many slots of like values, one CTA a (sequence, KV head): each element to the bounds of the short cases, and
    their mean to f32's and what roundings of 16-bit results leave of it.  All sequences see nearly the same means of the values,
    so 8 D roundings are independent, each of them even over [-u, u], of deviation u / sqrt(3); four deviations of their mean are
    4 u / sqrt(3 * 8 D)."""
    out, lse, want, want_lse = periodic(torch, ty, 8, 8, D, n, n_seq=80)
    u = HALF_STEP[ty] if ty != "f32" else 0.0
    assert torch.all((out - want).abs() <= u * want + 1.5 * F32_TOL)
    assert abs(float((out - want).mean())) <= 1.5 * F32_TOL + 4 * u / math.sqrt(24 * D) * float(want.mean())
    assert torch.all((lse - want_lse).abs() <= F32_TOL * want_lse)


@pytest.mark.parametrize("ty", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n", [32768, 262144])
@pytest.mark.parametrize("gap", [15.5, 25.05, 31.1])
def test_prompts_count_small_weights(torch, ty, n, gap):
    """The same for packed tokens behind a prefix, enough of them that one CTA takes all positions of its rows.  16-bit queries
    round each weight to half a step, here all of them alike.  O and l are f32 sums over n / 128 tiles, whose addends are all the
    same here: each sum rounds by up to 2^-24 of itself, and always to the same side, so O / l is off by up to 2 n / 128 of that."""
    got, want = one_above_many(torch, ty, n, gap, 1, tokens=2400)
    u = HALF_STEP[ty] if ty != "f32" else 0.0
    assert np.max(np.abs(got - want)) <= F32_TOL + 2 * (u + n / 128 * 2.0 ** -24) * want


@pytest.mark.parametrize("ty,n,kw", [
    ("f16", 131072, dict(tokens=2400, D=128)),              # row tiles of 256 behind a prefix
    ("bf16", 1048576, dict(tokens=2400, D=64)),
    ("f16", 131072, dict(n_seq=40, packed=True, D=128)),    # few rows: the positions of one row tile by both warpgroups
    ("bf16", 1048576, dict(n_seq=40, packed=True, D=64)),
    ("f16", 131072, dict(tokens=9000, D=64)),               # prefix and own slots by one item
    ("f32", 65536, dict(tokens=2400, D=128)),
    ("f32", 65536, dict(n_seq=40, packed=True, D=64)),
    ("f16", 8192, dict(tokens=2400, D=64)),                 # as many tiles as O takes at a time, and one more
    ("f16", 12288, dict(tokens=2400, D=128)),
])
def test_rows_over_long_ranges(torch, ty, n, kw):
    """Sums over many positions of like values on the tensor core: elements and their mean to the bounds of the single tokens'
    test, with half a step more for 16-bit weights."""
    out, lse, want, want_lse = periodic(torch, ty, 8, 8, n=n, **kw)
    u = HALF_STEP[ty] if ty != "f32" else 0.0
    assert torch.all((out - want).abs() <= 2 * u * want + 1.5 * F32_TOL)
    assert abs(float((out - want).mean())) <= 1.5 * F32_TOL + (u / 8 + 4 * u / math.sqrt(24 * kw["D"])) * float(want.mean())
    assert torch.all((lse - want_lse).abs() <= F32_TOL * want_lse)


@pytest.mark.parametrize("ty,D", [("f16", 128), ("bf16", 64), ("f32", 64)])
@pytest.mark.parametrize("prefix", [False, True])
def test_rows_whose_scores_climb_over_long_ranges(torch, ty, D, prefix):
    """25,600 positions whose keys grow by a factor of eight on the way: the running reference of the softmax moves after tiles of
    O have been put aside, too, and then they are rescaled with it."""
    from fish_s2pro_b200 import PagedKvCache
    G, n = 8, 25600
    gen = torch.Generator(device="cuda").manual_seed(D)
    kv = torch.bfloat16 if ty == "bf16" else torch.float16
    grow = 1.0 + 7.0 * torch.arange(n // PAGE, device="cuda") / (n // PAGE)
    k = (torch.randn(n // PAGE, G, PAGE, D, generator=gen, device="cuda") * grow[:, None, None, None]).to(kv)
    v = torch.randn(n // PAGE, G, PAGE, D, generator=gen, device="cuda").to(kv)
    ids = torch.arange(n // PAGE, device="cuda", dtype=torch.int32)
    T = 4800 if prefix else 40
    q = torch.randn(T, G, D, generator=gen, device="cuda").to(act_dtype(torch, ty))
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    if prefix:
        c = PagedKvCache(k, v, ints([[0]]), ints([0]))
        out = c.attention(q, q_start=ints([0, T]), prefix_pages=ids, prefix_len=n)
    else:
        c = PagedKvCache(k, v, ids.expand(T, -1).contiguous(), ints([n] * T))
        out = c.attention(q, q_start=ints(list(range(T + 1))))
    c.check()
    some = torch.arange(0, T, 97 if prefix else 1, device="cuda")
    rows = lambda x: x.permute(1, 0, 2, 3).reshape(G, -1, D).double()
    s = torch.einsum("tgd,gnd->tgn", q[some].double(), rows(k)) / math.sqrt(D)
    w = s.softmax(-1)
    want, spread = torch.einsum("tgn,gnd->tgd", w, rows(v)), torch.einsum("tgn,gnd->tgd", w, rows(v).abs())
    u = HALF_STEP[ty]
    # scores reach some tens: 2^-24 of them in an exponent, and the products' truncation (8 steps of 16 elements), 2^-20 of a weight
    bound = u * want.abs() + (u if ty != "f32" else 0) * spread + (2.0 ** -20 * float(s.abs().max()) * spread) + F32_TOL * float(v.abs().max())
    assert torch.all((out[some].double() - want).abs() <= bound)


def test_gains_that_require_a_gradient_are_refused(torch):
    """The gains are a model's parameters: with gradients on, the queries would be cut off from them.  Without, they are taken.
    The same for a cache of such tensors."""
    from fish_s2pro_b200 import PagedKvCache, S2dError
    s = Case(torch, "f16", 8, 2, 64, [30, 40], None, 0, seed=45)
    kn, gain = torch.ones(2, 2, 64, dtype=torch.float16, device="cuda"), torch.nn.Parameter(torch.full((64,), 2.0, device="cuda"))
    pos, past = s.ints([1, 2]), s.ints([3, 4])
    for kw in (dict(q_norm=gain), dict(k_norm=gain), dict(q_norm=gain, k_norm=gain.detach())):
        with pytest.raises(S2dError, match="gradient") as e:
            s.c.append(s.q, kn, kn, pos, past, **kw)
        assert e.value.code == -1
    want = s.c.append(s.q, kn, kn, pos, past, q_norm=gain.detach(), k_norm=gain.detach())
    with torch.no_grad():
        assert torch.equal(s.c.append(s.q, kn, kn, pos, past, q_norm=gain, k_norm=gain), want)
    s.c.check()
    k = s.c.k.clone().requires_grad_()
    for buffers in ((k, s.c.v), (s.c.k, k)):
        with pytest.raises(S2dError, match="gradient"):
            PagedKvCache(*buffers, s.c.page_table, s.c.lengths)


@pytest.mark.parametrize("end", [-1, -2 ** 31, -2 ** 31 + 40])
def test_append_of_starts_that_end_below_zero(torch, end):
    """A last entry so far below zero that its distance to a block's first token is no int: no row is read or written, whichever
    block it is (650 tokens: groups of two, the last of them past the tokens if it counted)."""
    from fish_s2pro_b200 import S2dError
    T = 651
    s = Case(torch, "f16", 8, 2, 64, [192, 192], [T - 200, 200], 0, seed=47)
    wide = torch.full((T + 40, 8, 64), 5.0, dtype=torch.float16, device="cuda")
    kn = torch.ones(T + 40, 2, 64, dtype=torch.float16, device="cuda")
    before = s.c.v.clone()
    s.c.append(s.q, kn[:T], kn[:T], s.ints([0] * T), s.ints([0, 0]), q_start=s.ints([0, 100, end]), out=wide[:T])
    with pytest.raises(S2dError, match="out of range"):
        s.c.check()
    assert torch.all(wide == 5.0) and torch.equal(s.c.v.view(torch.int16), before.view(torch.int16))


@pytest.mark.parametrize("prefix,n_seq", [(0, 3), (100, 3), (100, 300)])
def test_rows_before_the_first_sequence_stay(torch, prefix, n_seq):
    """q_start[0] above 0: reported by every call, and the rows below it, which are no sequence's, are left as they are, whether
    parts are joined or not; the sequences' rows come out as they should."""
    from fish_s2pro_b200 import S2dError
    s = Case(torch, "bf16", 8, 2, 64, [130, 150, 70] * (n_seq // 3), [20] * n_seq, prefix, seed=46)
    s.starts[0], s.tokens = 7, [13] + [20] * (n_seq - 1)
    s.q_start = s.ints(s.starts)
    out, lse = torch.full_like(s.q, 5.0), None
    got, lse = s.attend(out=out)
    assert torch.all(out[:7] == 5.0)
    with pytest.raises(S2dError, match="out of range"):
        s.c.check()
    want, want_lse, _, spread = s.expected()
    u = HALF_STEP["bf16"]
    assert np.all(np.abs(out.double().cpu().numpy() - want)[7:] <= (u * (np.abs(want) + spread) + F32_TOL * 8)[7:])
    assert np.all(np.abs(lse.double().cpu().numpy() - want_lse)[7:] <= F32_TOL * np.maximum(1, np.abs(want_lse[7:])))
    T = s.q.shape[0]
    kn = torch.randn(T, 2, 64, dtype=torch.bfloat16, device="cuda")
    q = torch.full_like(s.q, 5.0)
    past = torch.clamp(s.c.lengths - 40, min=0)
    s.c.append(s.q, kn, kn, s.ints([0] * T), past, q_start=s.q_start, out=q)  # position 0: the queries as they are
    with pytest.raises(S2dError, match="out of range"):
        s.c.check()
    assert torch.all(q[:7] == 5.0) and torch.equal(q[7:], s.q[7:])
    for b in (0, 1, n_seq - 1):
        at = [int(past[b]) + i for i in range(s.tokens[b])]
        rows = torch.stack([s.c.v[int(s.table[b, j // PAGE]), :, j % PAGE] for j in at])
        assert torch.equal(rows, kn[int(s.starts[b]): int(s.starts[b + 1])])
    assert s.c.lengths.tolist() == [int(p) + n for p, n in zip(past, s.tokens)]


class SharedPages:
    """Long tables at little memory: every sequence's row draws its pages from one small pool, which attention only reads.  The
    reference is the formula in float64 on the GPU, a sequence at a time."""

    def __init__(self, torch, ty, H, G, D, lengths, max_pages, tokens=None, prefix_len=0, pool=70, seed=0):
        from fish_s2pro_b200 import PagedKvCache
        gen = torch.Generator(device="cuda").manual_seed(seed)
        kv, B = torch.bfloat16 if ty == "bf16" else torch.float16, len(lengths)
        counts = [1] * B if tokens is None else tokens
        self.torch, self.ty, self.H, self.G, self.D, self.lengths, self.prefix_len = torch, ty, H, G, D, lengths, prefix_len
        self.starts = np.concatenate([[0], np.cumsum(counts)]).tolist()
        self.k, self.v = (torch.randn(pool, G, PAGE, D, generator=gen, device="cuda").to(kv) for _ in range(2))
        self.table = torch.randint(0, pool, (B, max_pages), generator=gen, device="cuda", dtype=torch.int32)
        self.prefix = torch.randint(0, pool, (-(-prefix_len // PAGE),), generator=gen, device="cuda", dtype=torch.int32)
        self.q = (torch.randn(self.starts[-1], H, D, generator=gen, device="cuda") * 2).to(act_dtype(torch, ty))
        self.mass0 = torch.rand(B, G, max_pages * PAGE, generator=gen, device="cuda")
        self.mass, self.scale = self.mass0.clone(), 1 / math.sqrt(D)
        ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
        self.c = PagedKvCache(self.k, self.v, self.table, ints(lengths), mass=self.mass)
        self.q_start = None if tokens is None else ints(self.starts)

    def check(self, weigh=True):
        torch, G, D, rep = self.torch, self.G, self.D, self.H // self.G
        out, lse = self.c.attention(self.q, q_start=self.q_start, prefix_pages=self.prefix if self.prefix_len else None,
                                    prefix_len=self.prefix_len, weigh=weigh, scale=self.scale, return_lse=True)
        self.c.check()
        u, want_mass, P = HALF_STEP[self.ty], self.mass0.double(), self.prefix_len
        rows = lambda x, pages, n: x[pages.long()].permute(1, 0, 2, 3).reshape(G, -1, D)[:, :n].double()
        most = float(self.v.abs().max())
        for b, n in enumerate(self.lengths):
            t0, t1 = self.starts[b], self.starts[b + 1]
            if t1 == t0:
                continue
            k, v = (torch.cat([rows(x, self.prefix, P), rows(x, self.table[b], n)], 1) for x in (self.k, self.v))
            s = torch.einsum("tgrd,gnd->tgrn", self.q[t0:t1].double().view(-1, G, rep, D), k) * self.scale
            last = P + (n - (t1 - t0) + torch.arange(t1 - t0, device="cuda")).clamp(min=-1)  # tokens without a slot see the prefix
            s.masked_fill_((torch.arange(P + n, device="cuda") > last[:, None])[:, None, None], -math.inf)
            w = torch.softmax(s, -1).nan_to_num(0.0)
            want, spread = torch.einsum("tgrn,gnd->tgrd", w, v), torch.einsum("tgrn,gnd->tgrd", w, v.abs())
            bound = u * want.abs() + (u if self.ty != "f32" else 0) * spread + F32_TOL * most
            assert torch.all((out[t0:t1].double().view(want.shape) - want).abs() <= bound), b
            want_lse, got = torch.logsumexp(s, -1), lse[t0:t1].double().view(s.shape[:-1])
            seen = want_lse > -math.inf
            assert torch.all((got - want_lse)[seen].abs() <= F32_TOL * want_lse[seen].abs().clamp(min=1)), b
            assert torch.all(got[~seen] == -math.inf)
            if weigh:
                want_mass[b, :, :n] += w[..., P:].sum((0, 2))
        assert torch.all((self.mass.double() - want_mass).abs() <= F32_TOL * want_mass.clamp(min=1))
        beyond = torch.arange(self.mass.shape[2], device="cuda") >= torch.tensor(self.lengths, device="cuda")[:, None, None]
        assert torch.all((self.mass == self.mass0) | ~beyond)


def ragged_lengths(n_seq, most, seed):
    rng = np.random.default_rng(seed)
    x = rng.integers(0, most + 1, n_seq)
    x[:4] = [most, 0, 1, most - 1]
    return x.tolist()


@pytest.mark.parametrize("ty,H,G,D,n_seq,max_pages,prefix", [
    ("f16", 32, 8, 128, 64, 128, 0),      # tables of 8,192 slots: more CTAs a sequence, so that two of them fit an SM
    ("f32", 32, 8, 128, 64, 128, 300),
    ("bf16", 32, 8, 128, 64, 100, 65),
    ("f16", 32, 8, 128, 80, 128, 0),      # one CTA a (sequence, KV head), which keeps up to 8,192 scores
    ("f32", 32, 8, 128, 80, 128, 200),
    ("bf16", 64, 8, 128, 80, 64, 300),    # eight heads a group: more outputs than threads, behind prefix parts
    ("f16", 64, 8, 64, 80, 64, 1000),
    ("f16", 8, 1, 128, 2, 606, 300),      # eight CTAs a sequence: the longest table whose scores fit, and a longer one
    ("f16", 8, 1, 128, 2, 608, 300),
    ("f32", 8, 1, 128, 1, 608, 0),
    ("bf16", 8, 1, 64, 2, 740, 0),
    ("f32", 8, 2, 64, 3, 1600, 130),      # weights from scores computed again
    ("f16", 32, 8, 128, 80, 170, 64),
    ("bf16", 32, 2, 128, 9, 40, 500),     # sixteen heads a group
])
def test_single_tokens_that_weigh_in_long_tables(torch, ty, H, G, D, n_seq, max_pages, prefix):
    lengths = ragged_lengths(n_seq, max_pages * PAGE, n_seq + max_pages) if n_seq > 3 else [max_pages * PAGE - 5, 700, 0][:n_seq]
    SharedPages(torch, ty, H, G, D, lengths, max_pages, prefix_len=prefix, seed=max_pages).check()


@pytest.mark.parametrize("ty", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("scale", [-0.125, 0.0, -0.0, 1e-30])
@pytest.mark.parametrize("tokens", [None, [3, 0, 151, 40]])
def test_negative_and_zero_scales(torch, ty, scale, tokens):
    """The maximum of scale * q . k where the scale is negative is the minimum of q . k; scale 0 weighs every position alike."""
    for H, G, D, prefix in ((8, 2, 64, 200), (32, 8, 128, 0), (16, 1, 128, 70)):
        s = SharedPages(torch, ty, H, G, D, [130, 700, 150, 64], 12, tokens, prefix, seed=D)
        s.scale = scale
        s.check()


def test_a_new_cache_on_another_stream(torch):
    """A cache made on a busy stream and used on another: its status word is clear there too, and what it reports is not cleared
    when the first stream gets that far."""
    from fish_s2pro_b200 import PagedKvCache, S2dError
    s = Case(torch, "f16", 8, 2, 64, [30, 40], None, 0, seed=48)
    bad = s.ints([30, -1])
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for lengths, fails in ((s.c.lengths, False), (bad, True)):
        trash = [torch.full((1,), -1, dtype=torch.int32, device="cuda") for _ in range(64)]  # what a new word may hold
        torch.cuda.synchronize()
        del trash
        torch.cuda._sleep(400_000_000)
        c = PagedKvCache(s.c.k, s.c.v, s.c.page_table, lengths)
        with torch.cuda.stream(side):
            c.attention(s.q)
            side.synchronize()
            torch.cuda.synchronize()
            if fails:
                with pytest.raises(S2dError, match="out of range"):
                    c.check()
            else:
                c.check()
    torch.cuda.synchronize()


def test_a_cache_made_while_capturing(torch):
    """A function that makes its cache can be captured: the word is cleared at each replay, and the results are the eager ones."""
    from fish_s2pro_b200 import PagedKvCache
    s = Case(torch, "f16", 8, 2, 64, [30, 40], None, 0, seed=49)
    want = PagedKvCache(s.c.k, s.c.v, s.c.page_table, s.c.lengths).attention(s.q)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        c = PagedKvCache(s.c.k, s.c.v, s.c.page_table, s.c.lengths)
        out = c.attention(s.q)
    g.replay()
    c.check()
    assert torch.equal(out, want)


def test_status_words_of_many_caches(torch):
    """Words come in blocks: what one cache reports no other does, past the end of a block too."""
    from fish_s2pro_b200 import PagedKvCache, S2dError
    s = Case(torch, "f16", 8, 2, 64, [30, 40], None, 0, seed=51)
    bad = s.ints([30, -1])
    caches = [PagedKvCache(s.c.k, s.c.v, s.c.page_table, bad if i % 500 == 7 else s.c.lengths) for i in range(1100)]
    for c in caches:
        c.attention(s.q)
    for i, c in enumerate(caches):
        if i % 500 == 7:
            with pytest.raises(S2dError, match="out of range"):
                c.check()
        c.check()


def test_check_while_capturing_is_refused(torch):
    """The check waits, which a capture cannot: it says so and leaves the capture as it is."""
    from fish_s2pro_b200 import S2dError
    s = Case(torch, "f16", 8, 2, 64, [30, 40], None, 70, seed=50)
    want, _ = s.attend()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out, lse = s.attend()
        with pytest.raises(S2dError, match="captur") as e:
            s.c.check()
        assert e.value.code == -1
    g.replay()
    s.c.check()
    assert torch.equal(out, want)


@pytest.mark.parametrize("ty,tokens", [("f32", None), ("bf16", [40, 3, 0, 130])])
def test_heads_apart_in_the_pool(torch, ty, tokens):
    """A pool laid out [page][head][K | V][64][D]: a head stride that is not the rows' size."""
    from fish_s2pro_b200 import PagedKvCache
    s = SharedPages(torch, ty, 8, 4, 64, [200, 3, 0, 150], 4, tokens, 100, seed=3)
    pool = torch.stack([s.k, s.v], 2)
    s.c = PagedKvCache(pool[:, :, 0], pool[:, :, 1], s.table, s.c.lengths, mass=s.mass)
    s.check()


@pytest.mark.parametrize("ty,H,G,tokens", [("f16", 1024, 1024, None), ("bf16", 600, 300, [60, 5])])
def test_many_kv_heads(torch, ty, H, G, tokens):
    SharedPages(torch, ty, H, G, 64, [100, 37], 3, tokens, 70, pool=8, seed=1).check()


@pytest.mark.parametrize("packed", [False, True])
def test_the_most_sequences(torch, packed):
    """65,535 sequences of up to a page, each with one token: appended, and weighed over what they hold."""
    from fish_s2pro_b200 import PagedKvCache
    B, G, D = 65535, 2, 64
    gen = torch.Generator(device="cuda").manual_seed(5)
    k, v = (torch.randn(B, G, PAGE, D, generator=gen, device="cuda").half() for _ in range(2))
    table = torch.randperm(B, generator=gen, device="cuda").to(torch.int32).view(B, 1)
    past = torch.randint(0, PAGE, (B,), generator=gen, device="cuda", dtype=torch.int32)
    lengths, mass = torch.zeros_like(past), torch.zeros(B, G, PAGE, device="cuda")
    q, kn, vn = (torch.randn(B, n, D, generator=gen, device="cuda").half() for n in (4, G, G))
    starts = torch.arange(B + 1, device="cuda", dtype=torch.int32) if packed else None
    c = PagedKvCache(k, v, table, lengths, mass=mass)
    qr = c.append(q, kn, vn, torch.zeros_like(past), past, q_start=starts)  # position 0: nothing turns
    at = table[:, 0].long()
    assert torch.equal(lengths, past + 1) and torch.equal(qr, q)
    assert torch.equal(k[at, :, past.long()], kn) and torch.equal(v[at, :, past.long()], vn)
    out, lse = c.attention(qr, q_start=starts, weigh=True, return_lse=True)
    c.check()
    for b0 in range(0, B, 8192):
        b = slice(b0, min(B, b0 + 8192))
        s = torch.einsum("bgrd,bgnd->bgrn", q[b].double().view(-1, G, 2, D), k[at[b]].double()) / math.sqrt(D)
        s.masked_fill_(torch.arange(PAGE, device="cuda") >= lengths[b][:, None, None, None], -math.inf)
        w = s.softmax(-1)
        rows = v[at[b]].double()
        want, spread = torch.einsum("bgrn,bgnd->bgrd", w, rows).view(-1, 4, D), torch.einsum("bgrn,bgnd->bgrd", w, rows.abs()).view(-1, 4, D)
        bound = HALF_STEP["f16"] * (want.abs() + spread) + F32_TOL * float(v.abs().max())
        assert torch.all((out[b].double() - want).abs() <= bound)
        assert torch.all((lse[b].double() - torch.logsumexp(s, -1).view(-1, 4)).abs() <= 6 * F32_TOL)  # of at most 6
        assert torch.all((mass[b].double() - w.sum(2)).abs() <= 2 * F32_TOL)


@pytest.mark.parametrize("n", [5, 1000, 1 << 20, 1 << 24])
@pytest.mark.parametrize("packed", [False, True])
def test_the_longest_tables(torch, n, packed):
    """Tables of 2^18 pages, hardly filled and full, which repeat 64 pages: the weights of a slot's copies are alike."""
    from fish_s2pro_b200 import PagedKvCache
    pages, D, H = 1 << 18, 64, 8
    gen = torch.Generator(device="cuda").manual_seed(6)
    k, v = (torch.randn(64, 1, PAGE, D, generator=gen, device="cuda").half() for _ in range(2))
    table = (torch.arange(pages, device="cuda") % 64).to(torch.int32).view(1, pages)
    q = torch.randn(1, H, D, generator=gen, device="cuda").half()
    mass = torch.zeros(1, 1, pages * PAGE, device="cuda")
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    c = PagedKvCache(k, v, table, ints([n]), mass=mass)
    out, lse = c.attention(q, q_start=ints([0, 1]) if packed else None, weigh=True, return_lse=True)
    c.check()
    period = min(n, 4096)
    s = (q[0].double() @ k.reshape(-1, D)[:period].double().T) / math.sqrt(D)
    w = s.softmax(-1)
    want, spread = w @ v.reshape(-1, D)[:period].double(), w @ v.reshape(-1, D)[:period].double().abs()
    bound = HALF_STEP["f16"] * (want.abs() + spread) + F32_TOL * float(v.abs().max())
    assert torch.all((out[0].double() - want).abs() <= bound)
    assert torch.all((lse[0].double() - torch.logsumexp(s, -1) - math.log(n / period)).abs() <= 20 * F32_TOL)  # of at most 20
    got = mass[0, 0, :n].double().view(-1, period) if n >= period else mass[0, 0, :n].double()[None]
    assert torch.all((got * (n // period) - w.sum(0)).abs() <= F32_TOL)
    assert torch.all(mass[0, 0, n:] == 0)


def test_replays_of_other_batches(torch):
    """A captured ragged call, replayed after the starts, the lengths and the queries have changed on the device: what an eager
    call of the same sizes gives, with fewer tokens than it was captured for."""
    s = SharedPages(torch, "bf16", 16, 8, 64, [300, 700, 130, 64], 12, [40, 7, 60, 0], 900, seed=52)
    first = [x.clone() for x in (s.q_start, s.c.lengths, s.q)]
    g = torch.cuda.CUDAGraph()
    s.check(weigh=False)  # and warm
    with torch.cuda.graph(g):
        out, lse = s.c.attention(s.q, q_start=s.q_start, prefix_pages=s.prefix, prefix_len=900, weigh=True, return_lse=True)
    for starts, lengths in (([0, 1, 50, 90, 107], [1, 600, 700, 17]), ([0, 0, 0, 100, 100], [5, 0, 768, 3]), ([0, 10, 20, 30, 40], [768] * 4)):
        s.q_start.copy_(torch.tensor(starts, dtype=torch.int32))
        s.c.lengths.copy_(torch.tensor(lengths, dtype=torch.int32))
        s.q.normal_()
        s.mass.copy_(s.mass0)
        out.fill_(5.0)
        g.replay()
        got = [out.clone(), lse.clone(), s.mass.clone()]
        s.mass.copy_(s.mass0)
        want = s.c.attention(s.q, q_start=s.q_start, prefix_pages=s.prefix, prefix_len=900, weigh=True, return_lse=True)
        n = starts[-1]
        assert torch.equal(got[0][:n], want[0][:n]) and torch.equal(got[1][:n], want[1][:n]) and torch.equal(got[2], s.mass)
        assert torch.all(got[0][n:] == 5.0)
        s.mass.copy_(s.mass0)
        s.starts, s.lengths = starts, lengths
        s.check()
    for x, y in zip((s.q_start, s.c.lengths, s.q), first):
        x.copy_(y)
    g.replay()
    s.c.check()
