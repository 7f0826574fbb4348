"""The cache in 4 bits on the GPU: cache_append_int4 and cache_read_int4 (whole
codes, against the oracle in 64 bits) and paged_attention_int4 (against the
formula in 64 bits over the values that the codes stand for).

Tolerances, derived: an output rounded once to a type of p significand bits
is off by at most u = 2^-p of its value (2^-11 FP16, 2^-8 BF16) plus half the
least subnormal; FP32 sums of n products by n 2^-24 of the sum of their
magnitudes.  A score sums head_dim products of the query with codes, then one
of scale and one of low a group: with r = sum |q| (15 |scale| + |low|) it is
off by d = (head_dim + 16) 2^-24 r |softmax scale|, which moves each weight by
at most 2 d relative.  Sums over n keys add n 2^-24, exponentials, quotients
and the weights' two FP16 parts less than 2^-20, all relative to sum p (15
|scale| + |low|)."""
import numpy as np
import pytest
import torch

from libortho_amd import _C_ops, _lib
from oracle import cache_oracle as O

pytestmark = pytest.mark.gpu

DT = {"fp16": torch.float16, "bf16": torch.bfloat16}
U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}
LAYOUTS = [(128, 128), (128, 64), (128, 32), (64, 64), (64, 32), (32, 32), (80, 80), (96, 96), (96, 32), (112, 112), (8, 8),
           (24, 24), (72, 72), (256, 256), (256, 128), (256, 64), (256, 32), (160, 32), (192, 64), (200, 200), (136, 136)]


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def np64(t):
    return t.double().cpu().numpy()


def random_cache(g, pages, P, G, D, group, dev="cuda"):
    """Codes and scales of normal vectors, quantised by the oracle's rules with torch for speed."""
    cache = []
    for _ in "kv":
        codes = torch.randint(0, 256, (pages, P, G, O.row_bytes(D)), generator=g, device=dev, dtype=torch.uint8)
        scales = torch.empty(pages, P, G, D // group, 2, dtype=torch.float16, device=dev)
        scales[..., 0] = torch.rand(scales.shape[:-1], generator=g, device=dev) * 0.3 + 0.05
        scales[..., 1] = -7.5 * scales[..., 0] + 0.3 * torch.randn(scales.shape[:-1], generator=g, device=dev)
        cache += [codes, scales]
    return cache


# --------------------------------------------------------------------- append

def append_inputs(T, H, G, D, group, P, dt, seed=0):
    g = torch.Generator(device="cuda").manual_seed(1000 * T + D + seed)
    qkv = torch.randn(T, H + 2 * G, D, generator=g, device="cuda").to(dt)
    pages = -(-T // P) + 3
    cache = random_cache(g, pages, P, G, D, group)
    slots = torch.randperm(pages * P, generator=g, device="cuda")[:T].contiguous()
    return qkv[:, :H], qkv[:, H:H + G], qkv[:, H + G:], cache, slots


def check_written(cache, before, slots, k, v, group, live=None):
    """Each slot's bytes and scales are the oracle's; all others as before."""
    D = k.shape[-1]
    live = list(range(len(slots))) if live is None else live
    at = [int(slots[i]) for i in live]
    for x, codes, scales, codes0, scales0 in ((k, *cache[:2], *before[:2]), (v, *cache[2:], *before[2:])):
        u, s, low = O.quantise(x[live], group)
        want_c, want_s = codes0.flatten(0, 1).cpu().numpy().copy(), scales0.flatten(0, 1).cpu().numpy().copy()
        want_c[at], want_s[at] = O.pack(u), np.stack([s, low], -1)
        np.testing.assert_array_equal(codes.flatten(0, 1).cpu().numpy(), want_c)
        np.testing.assert_array_equal(scales.flatten(0, 1).cpu().numpy(), want_s)


def check_turned(got, q, cs, pos, inter, dt):
    rot = cs.shape[1]
    rows = np64(cs)[pos.cpu().numpy()]
    want = O.turn(np64(q), rows[:, :rot // 2], rows[:, rot // 2:], inter)
    mag = O.turn(np.abs(np64(q)), np.abs(rows[:, :rot // 2]), -np.abs(rows[:, rot // 2:]), inter)
    mag = np.maximum(np.abs(mag), np.abs(O.turn(np.abs(np64(q)), np.abs(rows[:, :rot // 2]), np.abs(rows[:, rot // 2:]), inter)))
    err = np.abs(np64(got) - want)
    assert (err <= U[dt] * 1.01 * np.abs(want) + TINY[dt] + 2.0 ** -22 * mag).all(), err.max()


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("D,group", LAYOUTS)
def test_append_layouts(gpu, D, group, dtype):
    dt = DT[dtype]
    for T, H, G, rot, inter, P in [(5, 4, 2, D, False, 16), (3, 3, 3, D // 2 // 2 * 2, True, 5), (1, 2, 1, D // 2 // 2 * 2, False, 1)]:
        q, k, v, cache, slots = append_inputs(T, H, G, D, group, P, dt)
        before = [t.clone() for t in cache]
        pos = i32([(7 * t + 3) % 40 for t in range(T)])
        cs = torch.randn(41, rot, device="cuda")
        out = _C_ops.cache_append_int4(k, v, *cache, slots, q=q, positions=pos, cos_sin=cs, interleaved=inter)
        rows = np64(cs)[pos.cpu().numpy()]
        check_written(cache, before, slots, O.turn(np64(k), rows[:, :rot // 2], rows[:, rot // 2:], inter), np64(v), group)
        check_turned(out, q, cs, pos, inter, dt)


@pytest.mark.parametrize("T,H,G,D,group,rot,inter,P", [
    (1, 32, 32, 128, 32, 128, False, 16), (33, 8, 2, 64, 64, 64, True, 8), (300, 8, 1, 96, 32, 48, False, 13),
    (700, 14, 2, 256, 128, 128, False, 64), (2048, 2, 3, 128, 64, 128, False, 32), (40, 70, 1, 80, 80, 40, True, 7)])
def test_append_sizes(gpu, T, H, G, D, group, rot, inter, P):
    q, k, v, cache, slots = append_inputs(T, H, G, D, group, P, torch.float16)
    before = [t.clone() for t in cache]
    g = torch.Generator(device="cuda").manual_seed(T)
    pos = torch.randint(0, 500, (T,), generator=g, device="cuda", dtype=torch.int32)
    cs = torch.randn(500, rot, generator=g, device="cuda")
    q2 = q.clone()
    out = _C_ops.cache_append_int4(k, v, *cache, slots, q=q2, positions=pos, cos_sin=cs, interleaved=inter, q_out=q2)
    assert out.data_ptr() == q2.data_ptr()
    rows = np64(cs)[pos.cpu().numpy()]
    check_written(cache, before, slots, O.turn(np64(k), rows[:, :rot // 2], rows[:, rot // 2:], inter), np64(v), group)
    check_turned(out, q, cs, pos, inter, torch.float16)


def test_append_without_turning_and_tokens_that_are_not_written(gpu):
    q, k, v, cache, slots = append_inputs(6, 4, 2, 64, 32, 4, torch.bfloat16)
    before = [t.clone() for t in cache]
    slots[1], slots[4] = -1, cache[0].shape[0] * 4
    assert _C_ops.cache_append_int4(k, v, *cache, slots) is None
    check_written(cache, before, slots, np64(k), np64(v), 32, live=[0, 2, 3, 5])
    # positions outside the table: not written, q zero
    cache = [t.clone() for t in before]
    cs = torch.randn(9, 64, device="cuda")
    pos = i32([0, 8, 9, -1, 3, 2 ** 31 - 1])
    out = _C_ops.cache_append_int4(k, v, *cache, slots, q=q, positions=pos, cos_sin=cs)
    rows = np64(cs)[pos.cpu().numpy().clip(0, 8)]
    check_written(cache, before, slots, O.turn(np64(k), rows[:, :32], rows[:, 32:], False), np64(v), 32, live=[0])
    assert not bool(out[[2, 3, 5]].any()) and bool(out[4].any())
    # an empty table, no tokens
    cache = [t.clone() for t in before]
    out = _C_ops.cache_append_int4(k, v, *cache, slots, q=q, positions=pos, cos_sin=cs[:0])
    assert not bool(out.any()) and all(torch.equal(a, b) for a, b in zip(cache, before))
    assert _C_ops.cache_append_int4(k[:0], v[:0], *cache, slots[:0]) is None


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_append_numbers_at_the_edges(gpu, dtype):
    """Halves between two codes, ranges up to the type's ends, constants,
    subnormals, zeros of both signs, and groups that are not finite."""
    dt, D, group = DT[dtype], 128, 32
    rng = np.random.default_rng(3)
    rows = []
    for step in (1.0, 0.5, 2.0 ** -10, 3.0, 2.0 ** -24, 40.0):  # multiples of half a step, and their neighbours
        x = rng.integers(0, 31, D) * 0.5 * step
        x[::32], x[1::32] = 0, 15 * step
        rows += [x, -x, x + 7.5 * step, np.nextafter(x.astype(np.float16), np.float16(99)).astype(np.float64)]
    rows += [np.full(D, v) for v in (0.0, -0.0, 1.5, -65504.0, 65504.0, 2.0 ** -24)]
    wide = rng.uniform(-65504, 65504, D)
    wide[::32], wide[1::32] = -65504, 65504
    rows += [wide, np.abs(wide), -np.abs(wide), np.where(np.arange(D) % 2, 65504, 65472), rng.integers(-20, 21, D) * 2.0 ** -24]
    rows += [rng.standard_normal(D) * s for s in (1e-6, 1e-4, 300.0, 2e4)]
    for bad in (np.inf, -np.inf, np.nan):
        x = rng.standard_normal(D)
        x[37] = bad
        rows.append(x)
    if dtype == "bf16":
        rows += [rng.standard_normal(D) * s for s in (1e-30, 1e6, 1e38)]
    x = torch.tensor(np.array(rows)).to(dt).cuda()[:, None]
    T = x.shape[0]
    cache = list(_C_ops.int4_cache(T, 1, 1, D, group))
    before = [t.clone() for t in cache]
    slots = torch.arange(T, device="cuda").flip(0).contiguous()
    _C_ops.cache_append_int4(x, x.flip(0), *cache, slots)
    check_written(cache, before, slots, np64(x), np64(x.flip(0)), group)
    # turned: a quarter turn exchanges halves and their signs, and overflows nothing
    cs = torch.zeros(1, D, device="cuda")
    cs[:, D // 2:] = 1
    cache = [t.clone() for t in before]
    _C_ops.cache_append_int4(x, x, *cache, slots, positions=i32([0] * T), cos_sin=cs)
    with np.errstate(invalid="ignore"):
        want = O.turn(np64(x), np.zeros((T, D // 2)), np.ones((T, D // 2)), False)
    check_written(cache, before, slots, want, np64(x), group)


def test_append_strided_views_and_any_alignment(gpu):
    q, k, v, cache, slots = append_inputs(9, 4, 2, 64, 32, 8, torch.float16)
    cs, pos = torch.randn(60, 64, device="cuda"), i32([5 * t for t in range(9)])
    a, b = [t.clone() for t in cache], [t.clone() for t in cache]
    want = _C_ops.cache_append_int4(k, v, *a, slots, q=q, positions=pos, cos_sin=cs)
    # an odd element offset, heads outside tokens, keys and values of the cache side by side
    flat = torch.empty(3 * q.numel() + 1, dtype=torch.float16, device="cuda")[1:]
    k2 = flat[:k.numel()].view(2, 9, 64).transpose(0, 1)
    q2 = flat[2 * k.numel():2 * k.numel() + q.numel()].view(4, 9, 64).transpose(0, 1)
    k2.copy_(k)
    q2.copy_(q)
    codes, scales = torch.stack([b[0], b[2]], 1), torch.stack([b[1], b[3]], 1)
    got = _C_ops.cache_append_int4(k2, v, codes[:, 0], scales[:, 0], codes[:, 1], scales[:, 1], slots, q=q2, positions=pos, cos_sin=cs)
    assert torch.equal(got, want)
    for x, y in zip(a, (codes[:, 0], scales[:, 0], codes[:, 1], scales[:, 1])):
        assert torch.equal(x, y)


# ----------------------------------------------------------------------- read

def check_read(cache, slots, D, dt, **kw):
    k, v = _C_ops.cache_read_int4(*cache, slots, D, dt, **kw)
    n = cache[0].shape[0] * cache[0].shape[1]
    at = slots.cpu().numpy()
    ok = (at >= 0) & (at < n)
    for got, codes, scales in ((k, *cache[:2]), (v, *cache[2:])):
        val = O.values(codes.flatten(0, 1).cpu().numpy()[at.clip(0, n - 1)], scales.flatten(0, 1).cpu().numpy()[at.clip(0, n - 1)], D)
        want = np.where(ok[:, None, None], val, 0).astype(np.float32)  # (in FP32, then to the type: one rounding of 16 bits)
        assert torch.equal(got.cpu(), torch.from_numpy(want).to(dt)), (D, dt)
    return k, v


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("D,group", LAYOUTS)
def test_read_layouts(gpu, D, group, dtype):
    g = torch.Generator(device="cuda").manual_seed(D + group)
    for pages, P, G, n in ((3, 16, 2, 20), (5, 7, 3, 1), (2, 1, 1, 9), (40, 16, 5, 700)):
        cache = random_cache(g, pages, P, G, D, group)
        slots = torch.randint(-2, pages * P + 2, (n,), generator=g, device="cuda")
        check_read(cache, slots, D, DT[dtype])


def test_read_edges(gpu):
    g = torch.Generator(device="cuda").manual_seed(2)
    cache = random_cache(g, 4, 8, 2, 64, 32)
    k, v = check_read(cache, torch.tensor([2 ** 40, -2 ** 40, 2 ** 63 - 1, -2 ** 63, 31, 32], device="cuda"), 64, torch.float16)
    assert not bool(k[[0, 1, 2, 3, 5]].any()) and bool(k[4].any())
    k, v = _C_ops.cache_read_int4(*cache, torch.zeros(0, dtype=torch.int64, device="cuda"), 64)
    assert k.shape == v.shape == (0, 2, 64) and k.dtype == torch.float16
    # a scale that is not finite reads as NaN, in its group and slot alone
    cache[1][0, 3, 1, 1] = float("nan")
    k, _ = _C_ops.cache_read_int4(*cache, torch.arange(32, device="cuda"), 64, torch.bfloat16)
    bad = k.isnan()
    assert bool(bad[3, 1, 32:].all()) and int(bad.sum()) == 32
    # outputs in head order and at an odd offset
    slots = torch.arange(32, device="cuda").flip(0).contiguous()
    want = _C_ops.cache_read_int4(*cache, slots, 64)
    ko = torch.empty(2, 32, 64, dtype=torch.float16, device="cuda").transpose(0, 1)
    vo = torch.empty(32 * 2 * 64 + 1, dtype=torch.float16, device="cuda")[1:].view(32, 2, 64)
    k, v = _C_ops.cache_read_int4(*cache, slots, 64, k_out=ko, v_out=vo)
    assert k.data_ptr() == ko.data_ptr() and v.data_ptr() == vo.data_ptr()
    assert torch.equal(v, want[1]) and torch.equal(k.nan_to_num(), want[0].nan_to_num())


# ------------------------------------------------------------------ attention

def reference(q, cache, table, positions, rows, scale, window):
    """(out, bound) in 64 bits."""
    T, H, D = q.shape
    pages, P, G, _ = cache[0].shape
    dt, group = q.dtype, D // cache[1].shape[3]
    out, bound = np.zeros((T, H, D)), np.zeros((T, H, D))
    tab, (kc, ks, vc, vs) = table.cpu().numpy(), [t.cpu().numpy() for t in cache]
    qq = np64(q)
    held = {}
    for t in range(T):
        row, last = t if rows is None else int(rows[t]), int(positions[t])
        if last < 0 or row < 0 or row >= len(tab):
            continue
        if row not in held:
            pg = tab[row]
            ok = (pg >= 0) & (pg < pages)
            pg = np.where(ok, pg, 0)
            ok = np.repeat(ok, P)
            with np.errstate(invalid="ignore"):
                held[row] = [ok] + [O.values(c[pg].reshape(-1, G, c.shape[-1]), s[pg].reshape((-1, G) + s.shape[-2:]), D) for c, s in
                                    ((kc, ks), (vc, vs))] + \
                            [np.repeat(15 * np.abs(s[..., 0].astype(np.float64)) + np.abs(s[..., 1].astype(np.float64)), group, -1)
                             for s in (ks[pg].reshape((-1, G) + ks.shape[-2:]), vs[pg].reshape((-1, G) + vs.shape[-2:]))]
        ok, k, v, kr, vr = held[row]
        first = max(0, last + 1 - window) if window else 0
        j = np.arange(first, min(last + 1, len(ok)))
        j = j[ok[j]]
        if not len(j):
            continue
        for h in range(H):
            g = h // (H // G)
            with np.errstate(invalid="ignore"):
                s = k[j, g] @ qq[t, h] * scale
                d = (D + 16) * 2.0 ** -24 * float((kr[j, g] @ np.abs(qq[t, h])).max()) * abs(scale)
                p = np.exp(s - s.max())
                p /= p.sum()
                out[t, h] = p @ v[j, g]
                bound[t, h] = U[dt] * 1.01 * np.abs(out[t, h]) + TINY[dt] + (2 * d + 2.0 ** -20 + len(j) * 2.0 ** -24) * (p @ vr[j, g])
    return out, bound


def attend_case(lens, H, G, D, group, P, dt, seed=0, spare=3, width=None, sigma=2.0, new=1):
    g = torch.Generator(device="cuda").manual_seed(seed + D + P)
    counts = [-(-n // P) for n in lens]
    width = width or max(counts + [1]) + 1
    pages = sum(counts) + spare
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.full((len(lens), width), -1, dtype=torch.int32, device="cuda")
    at = 0
    for r, c in enumerate(counts):
        table[r, :c] = order[at:at + c]
        at += c
    q = (sigma * torch.randn(len(lens) * new, H, D, generator=g, device="cuda")).to(dt)
    return q, random_cache(g, pages, P, G, D, group), table, i32([n - new + i for n in lens for i in range(new)])


def attend_check(q, cache, table, pos, rows=None, scale=None, window=0, out=None):
    got = _C_ops.paged_attention_int4(q, *cache, table, pos, rows=rows, scale=scale, window=window, out=out)
    want, bound = reference(q, cache, table, pos, rows, q.shape[2] ** -0.5 if scale is None else scale, window)
    err = np.abs(np64(got) - want)
    assert (err <= bound).all(), (float((err - bound).max()), float(np.abs(want).max()), np.argwhere(~(err <= bound))[:3].tolist())
    return got


LENS = [0, 1, 2, 31, 32, 33, 64, 127, 129, 300, 513]


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("D,group", LAYOUTS)
def test_attention_layouts(gpu, D, group, dtype):
    attend_check(*attend_case(LENS, 4, 2, D, group, 16, DT[dtype]))


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("H,G,D,group,P", [
    (4, 4, 128, 32, 16), (8, 1, 64, 64, 8), (7, 1, 96, 32, 64), (16, 1, 128, 64, 16), (17, 1, 64, 32, 16), (40, 2, 128, 128, 128),
    (3, 3, 8, 8, 16), (4, 2, 72, 72, 24), (4, 4, 128, 64, 1), (8, 2, 64, 32, 7), (6, 2, 96, 96, 13), (5, 5, 248, 248, 20),
    (16, 1, 256, 32, 16), (32, 2, 160, 32, 8), (8, 2, 192, 64, 3), (64, 8, 128, 64, 32)])
def test_attention_heads_and_pages(gpu, H, G, D, group, P, dtype):
    attend_check(*attend_case(LENS, H, G, D, group, P, DT[dtype]))


@pytest.mark.parametrize("window", [1, 7, 32, 100, 1000])
@pytest.mark.parametrize("P", [16, 5])
def test_attention_window(gpu, window, P):
    attend_check(*attend_case(LENS, 4, 2, 128, 64, P, torch.float16), window=window)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("lens,H,G,D,group,P", [
    ([20000], 8, 2, 128, 64, 64), ([5000, 1, 0, 9001], 4, 4, 64, 32, 16), ([1, 7, 30000, 300, 2], 4, 1, 128, 128, 32),
    ([40] * 70 + [25000] + [3] * 20, 8, 4, 64, 64, 16), ([18000, 20000], 5, 1, 64, 32, 8), ([3000] * 3, 32, 4, 80, 80, 16),
    ([4097], 2, 1, 256, 64, 128)])
def test_attention_long(gpu, lens, H, G, D, group, P, dtype):
    attend_check(*attend_case(lens, H, G, D, group, P, DT[dtype]))


def test_attention_many_short_requests(gpu):
    rng = np.random.default_rng(5)
    attend_check(*attend_case(rng.integers(0, 60, 400).tolist(), 4, 2, 64, 64, 16, torch.bfloat16, width=40))


@pytest.mark.parametrize("H,G,D,group,P,window", [(8, 2, 128, 64, 16, 0), (4, 4, 64, 64, 16, 40), (8, 1, 128, 32, 5, 0),
                                                  (16, 1, 80, 80, 8, 3), (6, 2, 96, 32, 16, 33), (34, 2, 64, 32, 16, 0)])
@pytest.mark.parametrize("new", [1, 2, 3, 17, 40])
def test_attention_several_tokens_of_a_request(gpu, H, G, D, group, P, window, new):
    lens = [new, new + 1, 70, 500, 64 + new]
    q, cache, table, pos = attend_case(lens, H, G, D, group, P, torch.float16, new=new)
    rows = i32([r for r in range(len(lens)) for _ in range(new)])
    attend_check(q, cache, table, pos, rows=rows, window=window)


def test_attention_rows_in_any_order(gpu):
    # tokens of a prompt, padding, unknown rows, a request's tokens backwards and apart
    q, cache, table, _ = attend_case([70, 40, 90], 8, 2, 128, 32, 16, torch.float16)
    rows = i32([1, 1, 1, 0, -1, 2, 2, 3, 0, 2 ** 31 - 1, 2, 2, 2, 2, 0, 1, 2, 0, 0, 0, 0, 1, 1, 1, 1, -5])
    pos = i32([37, 38, 39, 69, -1, 0, 88, 4, -1, 3, 88, 60, 3, 1, 2, 1, 50, -1, -1, -1, 12, 2 ** 31 - 1, 6, 6, 6, 0])
    q = torch.randn(len(rows), 8, 128, device="cuda").half()
    for window in (0, 5):
        got = attend_check(q, cache, table, pos, rows=rows, window=window)
        assert bool((got[[4, 7, 8, 9, 17, 18, 19, 25]] == 0).all())


def test_attention_a_prompt_token_by_token_and_at_once(gpu):
    # the same keys in one call and in calls of one token each: close to the same formula,
    # and a later token's key that is NaN reaches no earlier token
    n = 50
    q, cache, table, pos = attend_case([200], 8, 2, 64, 32, 16, torch.bfloat16, new=n)
    rows = i32([0] * n)
    got = attend_check(q, cache, table, pos, rows=rows)
    last = 199
    page, at = int(table[0, last // 16]), last % 16
    for i in range(4):
        if i % 2:
            old = cache[i][page, at].clone()
            cache[i][page, at] = float("nan")
            again = _C_ops.paged_attention_int4(q, *cache, table, pos, rows=rows)
            assert torch.equal(again[:-1], got[:-1]) and bool(again[-1].isnan().all())
            cache[i][page, at] = old


def test_attention_hides_whatever_masked_places_hold(gpu):
    for P in (16, 24, 5):
        q, cache, table, pos = attend_case([5, 33, 100, 1], 4, 2, 128, 32, P, torch.float16)
        want = attend_check(q, cache, table, pos, window=30)
        seen = torch.zeros(cache[0].shape[0], P, dtype=torch.bool, device="cuda")
        for r, n in enumerate([5, 33, 100, 1]):
            for j in range(max(0, n - 30), n):
                seen[int(table[r, j // P]), j % P] = True
        for bad in (float("nan"), float("inf"), -65504.0):
            other = [t.clone() for t in cache]
            for i, t in enumerate(other):
                t[~seen] = 255 if i % 2 == 0 else bad
            assert torch.equal(_C_ops.paged_attention_int4(q, *other, table, pos, window=30), want)


def test_attention_pages_outside_the_cache_are_not_seen(gpu):
    q, cache, table, pos = attend_case([100, 100, 40], 4, 2, 64, 64, 16, torch.bfloat16)
    table[0, 2] = -1
    table[0, 4] = cache[0].shape[0]
    table[1, :] = 2 ** 31 - 1  # sees nothing
    pos[2] = 5000              # past the table
    got = attend_check(q, cache, table, pos)
    assert bool((got[1] == 0).all())
    # several tokens of one request, whose first keys lie outside
    q = torch.randn(6, 4, 64, device="cuda").bfloat16()
    table[0, 0] = -7
    got = attend_check(q, cache, table, i32([3, 15, 16, 17, 18, 99]), rows=i32([0] * 6))
    assert bool((got[:2] == 0).all()) and bool((got[2] != 0).any())


def test_attention_extreme_scores(gpu):
    q, cache, table, pos = attend_case([3, 200, 64], 4, 2, 64, 32, 16, torch.float16)
    attend_check(q, cache, table, pos, scale=0.0)       # uniform weights
    attend_check(q * 30, cache, table, pos, scale=1.0)  # one weight takes all
    attend_check(q, cache, table, pos, scale=-0.125)
    # scores ever growing: every key raises the running maximum
    n = 400
    q, cache, table, pos = attend_case([n], 2, 1, 64, 64, 16, torch.bfloat16)
    q.fill_(1.0)
    cache[0].zero_()
    for j in range(n):
        cache[1][int(table[0, j // 16]), j % 16, 0, 0, 1] = j / 8.0
    attend_check(q, cache, table, pos, scale=0.05)
    cache[1][..., 1] -= 100  # scores far below zero: exp of them alone would vanish
    attend_check(q, cache, table, pos, scale=1.0)


def test_attention_values_of_very_different_sizes(gpu):
    # keys whose scales differ by 2^20 and more, the largest of them with weights that vanish, and groups of one head
    for dt in (torch.float16, torch.bfloat16):
        q, cache, table, pos = attend_case([120, 300], 4, 2, 128, 32, 16, dt, sigma=1.0)
        g = torch.Generator(device="cuda").manual_seed(4)
        e = torch.randint(-12, 8, cache[3].shape[:3], generator=g, device="cuda")
        cache[3] *= (2.0 ** e)[..., None, None].half()
        attend_check(q, cache, table, pos)
        small = [t.clone() for t in cache]
        small[3][...] = 2.0 ** -14 * torch.rand(small[3].shape, generator=g, device="cuda")
        huge = int(table[1, 3])
        small[3][huge, 5] = 8000.0                       # one key's values past all others by 2^27 ...
        small[1][huge, 5, ..., 1] = 0
        small[0][huge, 5] = 0
        small[1][huge, 5, ..., 0] = 0
        q[...] = q.abs()
        small[1][..., 1] = small[1][..., 1].abs() + 20   # ... whose weight is 0 beside keys of large scores
        small[1][huge, 5, ..., 1] = -60000.0
        attend_check(q, small, table, pos, scale=1.0)
        groups = [t.clone() for t in cache]
        groups[3][..., 1, :] *= 2.0 ** -13
        groups[3][..., 2, :] = 0                          # constants of zero
        groups[3][..., 3, 0] = 0                          # constants
        attend_check(q, groups, table, pos)


def test_attention_queries_of_any_size(gpu):
    for dt, sizes in ((torch.float16, (2.0 ** -20, 2.0 ** -10, 1.0, 3000.0)), (torch.bfloat16, (1e-37, 1e-20, 1e-5, 1e15, 1e30))):
        q, cache, table, pos = attend_case([1, 40, 333], 8, 2, 64, 64, 16, dt, sigma=1.0)
        for s in sizes:
            big = (q.float() * s).to(dt)
            attend_check(big, cache, table, pos, scale=0.1 / s)
        # elements of very different sizes in one query
        attend_check((q.float() * 2.0 ** torch.randint(-12, 3, q.shape, device="cuda")).to(dt), cache, table, pos)
        # one that is not finite, or NaN: its own heads' outputs are NaN
        for bad in (float("inf"), -float("inf"), float("nan")):
            x = q.clone()
            x[1, 3, 9] = bad
            out = _C_ops.paged_attention_int4(x, *cache, table, pos)
            assert bool(out[1, 3].isnan().all()) and int(out.isnan().sum()) == 64
        zero = torch.zeros_like(q)
        attend_check(zero, cache, table, pos)


def test_attention_groups_that_are_not_finite(gpu):
    q, cache, table, pos = attend_case([64, 64], 4, 2, 128, 32, 16, torch.float16)
    want = attend_check(q, cache, table, pos)
    a = [t.clone() for t in cache]
    a[3][int(table[1, 2]), 3, 1, 2] = float("nan")  # a value's group of one key head
    out = _C_ops.paged_attention_int4(q, *a, table, pos)
    assert bool(out[1, 2:, 64:96].isnan().all()) and int(out.isnan().sum()) == 2 * 32
    same = torch.ones_like(out, dtype=torch.bool)
    same[1, 2:] = False
    assert torch.equal(out[same], want[same])
    a = [t.clone() for t in cache]
    a[1][int(table[0, 0]), 3, 0, 2] = float("nan")  # a key's
    out = _C_ops.paged_attention_int4(q, *a, table, pos)
    assert bool(out[0, :2].isnan().all()) and int(out.isnan().sum()) == 2 * 128


def test_attention_strided_views(gpu):
    q, cache, table, pos = attend_case(LENS, 6, 3, 64, 32, 16, torch.float16)
    want = attend_check(q, cache, table, pos)
    wide = torch.randn(len(LENS), 20, 64, device="cuda").half()
    wide[:, 3:9] = q
    codes, scales = torch.stack([cache[0], cache[2]], 1), torch.stack([cache[1], cache[3]], 3)
    t2 = torch.zeros(len(LENS), table.shape[1] + 9, dtype=torch.int32, device="cuda")
    t2[:, :table.shape[1]] = table
    out = torch.empty(6, len(LENS), 64, dtype=torch.float16, device="cuda").transpose(0, 1)
    got = _C_ops.paged_attention_int4(wide[:, 3:9], codes[:, 0], scales[:, :, :, 0], codes[:, 1], scales[:, :, :, 1],
                                      t2[:, :table.shape[1]], pos, out=out)
    assert got.data_ptr() == out.data_ptr() and torch.equal(got, want)
    # heads outside slots, and an odd element offset of q and out
    head_major = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in cache]
    flat = torch.empty(2 * q.numel() + 1, dtype=torch.float16, device="cuda")[1:]
    q2, out2 = flat[:q.numel()].view(q.shape), flat[q.numel():].view(q.shape)
    q2.copy_(q)
    assert torch.equal(_C_ops.paged_attention_int4(q2, *head_major, table, pos, out=out2), want)


def test_attention_past_32_bit_offsets(gpu):
    # a cache of 2^32 + bytes of codes and 2^31 + of scales, the request's pages at its end
    P, G, D, group = 16, 4, 128, 32
    pages = (1 << 32) // (P * G * 64) + 40
    codes = torch.empty(pages, P, G, 64, dtype=torch.uint8, device="cuda")
    scales = torch.empty(pages, P, G, 4, 2, dtype=torch.float16, device="cuda")
    small = random_cache(torch.Generator(device="cuda").manual_seed(1), 40, P, G, D, group)
    codes[-40:], scales[-40:] = small[0], small[1]
    cache = [codes, scales, codes, scales]
    table = (pages - 1 - torch.arange(30, device="cuda", dtype=torch.int32))[None].contiguous()
    q = torch.randn(1, 8, D, device="cuda").half()
    got = _C_ops.paged_attention_int4(q, *cache, table, i32([450]))
    t40 = (39 - torch.arange(30, device="cuda", dtype=torch.int32))[None].contiguous()
    assert torch.equal(got, attend_check(q, [small[0], small[1], small[0], small[1]], t40, i32([450])))
    # and a slot written and read there
    k = torch.randn(1, G, D, device="cuda").half()
    slot = torch.tensor([pages * P - 3], device="cuda")
    _C_ops.cache_append_int4(k, k, *cache, slot)
    u, s, low = O.quantise(np64(k), group)
    assert np.array_equal(codes[-1, P - 3].cpu().numpy(), O.pack(u)[0])
    a, b = _C_ops.cache_read_int4(*cache, slot, D)
    assert torch.equal(a, b) and float((a - k).abs().max()) <= float(s.max())


@pytest.mark.parametrize("P", [32, 28])
def test_attention_last_key_numbers(gpu, P):
    # windows at the end of the widest table there is (one page in every place)
    W = ((1 << 31) - 512) // P
    table = torch.zeros(1, W, dtype=torch.int32, device="cuda")
    cache = random_cache(torch.Generator(device="cuda").manual_seed(P), 1, P, 1, 8, 8)
    q = torch.randn(1, 2, 8, device="cuda").half()
    k, v = (torch.from_numpy(O.values(cache[i].cpu().numpy(), cache[i + 1].cpu().numpy(), 8))[0, :, 0] for i in (0, 2))
    for back, window in ((1, 1), (1, 300), (40, 1000), (0, 70)):
        last = W * P - back  # (back 0: one key past the table, not seen)
        got = _C_ops.paged_attention_int4(q, *cache, table, i32([last]), window=window)
        j = torch.from_numpy(np.arange(max(0, last + 1 - window), min(last + 1, W * P)) % P)
        want = torch.softmax(q[0].double().cpu() @ k[j].T * 8 ** -0.5, -1) @ v[j]
        # FP16's rounding of values up to |v| <= 8, and FP32 sums behind it
        assert float((got[0].double().cpu() - want).abs().max()) <= 2 ** -8


def test_the_same_every_time_and_on_other_streams(gpu):
    q, cache, table, pos = attend_case([9000, 17, 4000], 8, 2, 128, 64, 16, torch.bfloat16)
    want = attend_check(q, cache, table, pos)
    slots = torch.arange(500, device="cuda")
    kv = _C_ops.cache_read_int4(*cache, slots, 128)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        assert torch.equal(_C_ops.paged_attention_int4(q, *cache, table, pos), want)
        with torch.cuda.stream(s):
            got = _C_ops.paged_attention_int4(q, *cache, table, pos)
            kv2 = _C_ops.cache_read_int4(*cache, slots, 128)
        s.synchronize()
        assert torch.equal(got, want) and torch.equal(kv2[0], kv[0]) and torch.equal(kv2[1], kv[1])


# ----------------------------------------------------------------- together

def test_step_append_attend_read_captured_and_replayed(gpu):
    """A serving step in a graph: replayed with other lengths and contents,
    each time the eager result."""
    P, W, H, G, D, T, group = 16, 40, 8, 2, 64, 6, 32
    g = torch.Generator(device="cuda").manual_seed(8)
    lengths, new = i32([0, 5, 100, 37]), i32([3, 1, 1, 1])
    table = torch.zeros(4, W, dtype=torch.int32, device="cuda")
    free = torch.randperm(120, generator=g, device="cuda").to(torch.int32)
    pool = i32([0, 0])
    cache = random_cache(g, 120, P, G, D, group)
    qkv = torch.randn(T, H + 2 * G, D, generator=g, device="cuda").half()
    cs = torch.randn(1000, D, generator=g, device="cuda")

    def step():
        L, p, _, rows, pos, slots = _C_ops.page_step(lengths, new, table, free, pool, P, T)
        q = _C_ops.cache_append_int4(qkv[:, H:H + G], qkv[:, H + G:], *cache, slots, q=qkv[:, :H], positions=pos, cos_sin=cs)
        return (_C_ops.paged_attention_int4(q, *cache, table, pos, rows=rows), L, p, *_C_ops.cache_read_int4(*cache, slots, D))

    for r, n in enumerate(lengths.tolist()):
        for j in range(-(-n // P)):
            table[r, j] = 119 - 10 * r - j
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for i in range(4):
        qkv.copy_(torch.randn(qkv.shape, generator=g, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in outs]
        for a, b in zip(got, step()):
            assert torch.equal(a, b), i
        attend_check(*attend_case([5, 40], 4, 2, 64, 32, 16, torch.float16))
        new.copy_(i32([[1, 1, 1, 1], [0, 2, 0, 3], [2, 2, 1, 1], [6, 0, 0, 0]][i]))


def test_a_cache_grown_token_by_token(gpu):
    """Prompts and single tokens through step, append and attention, against
    the formula over the oracle's own quantised keys and values."""
    P, H, G, D, group = 8, 6, 2, 96, 32
    g = torch.Generator(device="cuda").manual_seed(11)
    cache = list(_C_ops.int4_cache(60, P, G, D, group))
    table = torch.zeros(3, 20, dtype=torch.int32, device="cuda")
    lengths, pool = i32([0, 0, 0]), i32([0, 0])
    free = torch.randperm(60, generator=g, device="cuda").to(torch.int32)
    angle = torch.arange(160, device="cuda", dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, D, 2, device="cuda", dtype=torch.float64) / D)
    cs = torch.cat([angle.cos(), angle.sin()], 1).float().contiguous()
    keys, vals = [[], [], []], [[], [], []]
    for new in ([40, 0, 9], [1, 17, 1], [1, 1, 1], [0, 1, 5], [1, 1, 1]):
        T = sum(new)
        qkv = torch.randn(T, H + 2 * G, D, generator=g, device="cuda").half()
        lengths, pool, _, rows, pos, slots = _C_ops.page_step(lengths, i32(new), table, free, pool, P, T)
        q = _C_ops.cache_append_int4(qkv[:, H:H + G], qkv[:, H + G:], *cache, slots, q=qkv[:, :H], positions=pos, cos_sin=cs)
        out = attend_check(q, cache, table, pos, rows=rows)
        angles = np64(cs)[pos.cpu().numpy()]
        k = O.turn(np64(qkv[:, H:H + G]), angles[:, :D // 2], angles[:, D // 2:], False)
        for t, r in enumerate(rows.tolist()):
            for x, held in ((k[t], keys), (np64(qkv[t, H + G:]), vals)):
                u, s, low = O.quantise(x, group)
                held[r].append(np.repeat(low.astype(np.float64), group, -1) + u * np.repeat(s.astype(np.float64), group, -1))
        for r in range(3):
            n = int(lengths[r])
            assert len(keys[r]) == n
            if not n:
                continue
            j = torch.arange(n, device="cuda")
            a, b = _C_ops.cache_read_int4(*cache, table[r].long()[j // P] * P + j % P, D)
            for got, held in ((a, keys[r]), (b, vals[r])):
                assert torch.equal(got.cpu(), torch.from_numpy(np.array(held).astype(np.float32)).half())


# ------------------------------------------------------------------- refusals

def test_refusals(gpu):
    q, cache, table, pos = attend_case([5, 9], 4, 2, 64, 32, 16, torch.float16)
    kc, ks, vc, vs = cache
    A = _C_ops.paged_attention_int4
    for args, msg in [
            ((q.cpu(), *cache, table, pos), "device"), ((q.float(), *cache, table, pos), "float16 or bfloat16"),
            ((q, kc.int(), ks, vc, vs, table, pos), "codes"), ((q, kc, ks.float(), vc, vs, table, pos), "scales"),
            ((q, kc, ks, vc, vs[:, :, :, :1], table, pos), "scales"), ((q, kc, ks, vc[:1], vs, table, pos), "codes"),
            ((q, kc[..., :16], ks, vc[..., :16], vs, table, pos), "codes"), ((q[..., :60], *cache, table, pos), "head_dim"),
            ((q, kc.cpu(), ks, vc, vs, table, pos), "GPU"), ((q, kc, ks.transpose(3, 4), vc, vs.transpose(3, 4), table, pos), "scales"),
            ((q[:, :3], *cache, table, pos), "multiple of kv_heads"), ((q, *cache, table.long(), pos), "block_table"),
            ((q, *cache, table, pos.long()), "positions"), ((q, *cache, table[:1], pos), "rows of block_table"),
            ((q, *cache, table, pos[:1]), "positions"), ((q[0], *cache, table, pos), "tokens")]:
        with pytest.raises(RuntimeError, match=msg):
            A(*args)
    with pytest.raises(RuntimeError, match="window"):
        A(q, *cache, table, pos, window=-1)
    with pytest.raises(RuntimeError, match="out"):
        A(q, *cache, table, pos, out=q[:, :2])
    with pytest.raises(RuntimeError, match="overlap"):
        A(q, *cache, table, pos, out=q[:, :1].expand(2, 4, 64))
    odd = torch.zeros(kc.numel() + 16, dtype=torch.uint8, device="cuda")[1:1 + kc.numel()].view(kc.shape)
    with pytest.raises(RuntimeError, match="16-byte"):
        A(q, odd, ks, vc, vs, table, pos)
    half = torch.zeros(ks.numel() + 8, dtype=torch.float16, device="cuda")[1:1 + ks.numel()].view(ks.shape)
    with pytest.raises(RuntimeError, match="4-byte"):
        A(q, kc, half, vc, vs, table, pos)
    with pytest.raises(RuntimeError, match="group_size"):  # groups of 16
        wide = torch.zeros(*ks.shape[:3], 4, 2, dtype=torch.float16, device="cuda")
        A(q, kc, wide, vc, wide, table, pos)
    k, slots = torch.zeros(2, 2, 64, dtype=torch.float16, device="cuda"), torch.zeros(2, dtype=torch.int64, device="cuda")
    cs = torch.zeros(4, 64, device="cuda")
    for args, kw, msg in [
            ((k, k, *cache, slots.int()), {}, "slots"), ((k[:, :1], k, *cache, slots), {}, "kv_heads"),
            ((k.bfloat16(), k, *cache, slots), {}, "dtype"), ((k.float(), k.float(), *cache, slots), {}, "float16 or bfloat16"),
            ((k, k, *cache, slots), {"q": q}, "cos_sin"), ((k[0], k, *cache, slots), {}, "tokens"),
            ((k, k, *cache, slots), {"cos_sin": cs}, "positions"),
            ((k, k, *cache, slots), {"cos_sin": cs[:, :63].contiguous(), "positions": pos}, "rot"),
            ((k, k, *cache, slots), {"q": q, "cos_sin": cs, "positions": pos, "q_out": q[:, :2]}, "q_out"),
            ((k, k, *cache, slots), {"q_out": q}, "q_out")]:
        with pytest.raises(RuntimeError, match=msg):
            _C_ops.cache_append_int4(*args, **kw)
    for args, kw, msg in [
            ((*cache, slots.int(), 64), {}, "slots"), ((*cache, slots, 60), {}, "head_dim"), ((*cache, slots, 128), {}, "codes"),
            ((*cache, slots, 64, torch.float32), {}, "dtype"), ((*cache, slots, 64), {"k_out": k[:1]}, "k_out"),
            ((*cache, slots, 64), {"v_out": k.bfloat16()}, "v_out"), ((*cache, slots, 64), {"v_out": k[:, :1]}, "v_out"),
            ((*cache, slots, 64), {"v_out": k[:, :1].expand(2, 2, 64)}, "overlap")]:
        with pytest.raises(RuntimeError, match=msg):
            _C_ops.cache_read_int4(*args, **kw)


@pytest.mark.parametrize("binding", ["compiled", "ctypes"])
def test_no_gradient_is_lost_without_a_word(gpu, monkeypatch, binding):
    if binding == "ctypes":
        monkeypatch.setattr(_lib, "torch_ops", lambda: None)
    q, cache, table, pos = attend_case([5, 9], 4, 2, 64, 32, 16, torch.float16)
    names = dict(zip(("k_codes", "k_scales", "v_codes", "v_scales"), cache))
    k, slots = torch.randn(2, 2, 64, device="cuda").half(), torch.zeros(2, dtype=torch.int64, device="cuda")
    cs = torch.randn(20, 64, device="cuda")
    for f, kw, takes in (
            (_C_ops.paged_attention_int4, dict(q=q, block_table=table, positions=pos, out=torch.empty_like(q)), ["q", "k_scales", "v_scales", "out"]),
            (_C_ops.cache_append_int4, dict(k=k, v=k, slots=slots, q=q, positions=pos, cos_sin=cs, q_out=torch.empty_like(q)),
             ["k", "v", "k_scales", "v_scales", "q", "cos_sin", "q_out"]),
            (_C_ops.cache_read_int4, dict(slots=slots, head_dim=64, k_out=torch.empty_like(k), v_out=torch.empty_like(k)),
             ["k_scales", "v_scales", "k_out", "v_out"])):
        for t in takes:
            args = {n: (x.detach().clone() if torch.is_tensor(x) else x) for n, x in {**names, **kw}.items()}
            args[t].requires_grad_()
            with pytest.raises(RuntimeError, match=f"has no gradient.*{t} "):
                f(**args)
            with torch.no_grad():
                f(**args)


def test_ctypes_binding_gives_the_same(gpu, monkeypatch):
    q, cache, table, pos = attend_case(LENS, 4, 2, 64, 32, 16, torch.float16)
    k = torch.randn(len(LENS), 2, 64, device="cuda").half()
    slots, cs = torch.arange(len(LENS), device="cuda"), torch.randn(600, 64, device="cuda")

    def calls():
        c = [t.clone() for t in cache]
        turned = _C_ops.cache_append_int4(k, k, *c, slots, q=q, positions=pos, cos_sin=cs)
        return [turned, *c, *_C_ops.cache_read_int4(*c, slots, 64, torch.bfloat16), _C_ops.paged_attention_int4(q, *c, table, pos, window=50)]

    a = calls()
    monkeypatch.setattr(_lib, "torch_ops", lambda: None)
    for x, y in zip(a, calls()):
        assert torch.equal(x, y)
    test_refusals(gpu)
