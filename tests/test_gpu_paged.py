"""The paged cache's operators on the GPU: page_step (whole numbers, against a
request-by-request reference), cache_append and paged_attention (against the
formulas in 64 bits).

Tolerances, derived: an output rounded once to a type of p significand bits
is off by at most u = 2^-p of its value (2^-11 FP16, 2^-8 BF16) plus half the
least subnormal; FP32 sums of n products by n 2^-24 of the sum of their
magnitudes.  For attention a score error d moves each weight by at most 2 d
relative, exponentials and quotients add less than 2^-20, and weights split
in two 16-bit parts 2^-15 at most, all relative to sum p |v|."""
import numpy as np
import pytest
import torch

from libortho_amd import _C_ops, _lib

pytestmark = pytest.mark.gpu

DT = {"fp16": torch.float16, "bf16": torch.bfloat16}
U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


# ------------------------------------------------------------------ page step

def step_reference(lengths, new, table, free, head, P, tokens):
    table = [list(r) for r in table]
    F, W = len(free), len(table[0]) if table else 0
    out, start, status, at, used = list(lengths), [], 0, 0, head
    off = head
    rows, pos, slots = [-1] * tokens, [-1] * tokens, [-1] * tokens
    for r, (L, n) in enumerate(zip(lengths, new)):
        start.append(min(at, tokens))
        places = max(n, 0)
        room = L >= 0 and n >= 0 and L + n <= 2 ** 31 - 1 and at + places <= tokens and \
            (n == 0 or -(-(L + n) // P) <= W)
        need = -(-(L + n) // P) - -(-L // P) if room else 0
        granted = room and (need == 0 or off + need <= F)
        if granted:
            out[r] = L + n
            for j in range(need):
                table[r][-(-L // P) + j] = free[off + j]
            used = max(used, off + need) if need else used
        else:
            status |= 1 if not room else 2
        off += need
        for i in range(min(places, max(0, tokens - at))):
            rows[at + i] = r
            if granted:
                pos[at + i] = L + i
                slots[at + i] = table[r][(L + i) // P] * P + (L + i) % P
        at += places
    return out, [used, status], start + [min(at, tokens)], rows, pos, slots, table


def step_check(lengths, new, P, tokens=None, width=None, spare=7, head=0, free=None):
    rng = np.random.default_rng(len(lengths) * 31 + P)
    R = len(lengths)
    width = width if width is not None else max([-(-(max(L, 0) + max(n, 0)) // P) for L, n in zip(lengths, new)] + [1]) + 1
    counts = [min(width, -(-max(L, 0) // P)) for L in lengths]
    need = sum(max(0, -(-(L + n) // P) - -(-L // P)) for L, n in zip(lengths, new) if L >= 0 and n >= 0 and n < 10 ** 6)
    free = need + spare if free is None else free
    ids = rng.permutation(sum(counts) + free + head).astype(np.int32)
    table = np.full((R, width), -5, np.int32)
    at = 0
    for r, c in enumerate(counts):
        table[r, :c] = ids[at:at + c]
        at += c
    frees = ids[at:]
    tokens = sum(max(n, 0) for n in new) if tokens is None else tokens
    want = step_reference(lengths, new, table.tolist(), frees.tolist(), head, P, tokens)
    t = torch.full((R, width + 3), 99, dtype=torch.int32, device="cuda")
    t[:, :width] = torch.from_numpy(table).cuda()
    for again in range(2):  # the inputs stay: a repeated call gives the same
        got = _C_ops.page_step(i32(lengths), i32(new), t[:, :width], torch.from_numpy(frees.copy()).cuda(),
                               i32([head, 77]), P, tokens)
        for name, g, w in zip(("lengths", "pool", "query_start", "rows", "positions", "slots"), got, want):
            assert g.tolist() == w, (name, again)
        assert t[:, :width].tolist() == want[6] if R else True
        assert bool((t[:, width:] == 99).all())
    return want


@pytest.mark.parametrize("P", [1, 3, 16, 64])
@pytest.mark.parametrize("R", [1, 2, 63, 64, 65, 1000, 1025, 2100])
def test_page_step_mixed_requests(gpu, R, P):
    rng = np.random.default_rng(R + P)
    lengths = np.where(rng.random(R) < 0.2, 0, rng.integers(1, 300, R)).tolist()
    new = np.where(rng.random(R) < 0.2, rng.integers(0, 60, R), 1).tolist()
    want = step_check(lengths, new, P, head=5)
    assert want[1][1] == 0


def test_page_step_page_edges(gpu):
    for P in (1, 2, 16):
        step_check([0, 1, P - 1, P, P + 1, 2 * P], [0] * 6, P)
        step_check([0, 1, P - 1, P, P + 1, 2 * P], [1] * 6, P)
        step_check([0, 1, P - 1, P, P + 1, 2 * P], [P, P, P + 1, P - 1, 3 * P, 0], P)


def test_page_step_unused_places_and_empty(gpu):
    step_check([4, 0, 9], [1, 3, 1], 4, tokens=40)
    step_check([], [], 4, tokens=5, width=1)
    step_check([], [], 4, tokens=0, width=1)
    step_check([3, 2], [0, 0], 4, tokens=0)


def test_page_step_refusals_on_the_device(gpu):
    # out of pages: the second and every later request that needs one
    want = step_check([0, 0, 5, 3, 0], [8, 8, 1, 1, 4], 4, free=3)
    assert want[1] == [2, 2] and want[0] == [8, 0, 6, 4, 0]
    # past the table, out of places, negative numbers, past 2^31
    assert step_check([0, 5], [40, 1], 4, width=3)[1][1] == 1
    assert step_check([0, 5, 1], [6, 4, 1], 4, tokens=8)[1][1] == 1
    assert step_check([-3, 5, 2], [1, -2, 1], 4)[1][1] == 1
    assert step_check([2 ** 31 - 1, 5], [1, 1], 4, width=8)[1][1] == 1
    assert step_check([5, 5], [2 ** 31 - 1, 1], 4, width=8, tokens=6, free=9)[1][1] == 1


def test_page_step_at_its_most_requests(gpu):
    R = 8192
    want = step_check([r % 50 for r in range(R)], [1 + (r % 5 == 0) for r in range(R)], 16)
    assert want[1][1] == 0
    with pytest.raises(_lib.OrthoError, match="8192"):
        z = torch.zeros(R + 1, dtype=torch.int32, device="cuda")
        _C_ops.page_step(z, z, torch.zeros(R + 1, 1, dtype=torch.int32, device="cuda"), z, i32([0, 0]), 16, 0)


# --------------------------------------------------------------- cache append

def turned(x, cos_sin, positions, interleaved):
    """(turned x, the sum of magnitudes behind each element) in 64 bits."""
    x = x.double().cpu().clone()
    mag = x.abs()
    rot = cos_sin.shape[1]
    rows = cos_sin.double().cpu()[positions.cpu().long().clamp(0, max(0, cos_sin.shape[0] - 1))]
    for i in range(rot // 2):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)
        c, s = rows[:, i, None], rows[:, rot // 2 + i, None]
        u, w = x[..., a].clone(), x[..., b].clone()
        x[..., a], x[..., b] = u * c - w * s, w * c + u * s
        mag[..., a], mag[..., b] = (u * c).abs() + (w * s).abs(), (w * c).abs() + (u * s).abs()
    return x, mag


def close(got, want, mag, dtype):
    err = (got.double().cpu() - want).abs()
    bound = U[dtype] * 1.01 * want.abs() + TINY[dtype] + 2.0 ** -22 * mag
    assert bool((err <= bound).all()), float((err - bound).max())


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("T,H,G,D,rot,inter,P", [
    (1, 32, 32, 128, 128, False, 16), (5, 8, 2, 64, 64, True, 8), (33, 4, 4, 80, 40, False, 16),
    (7, 6, 3, 112, 56, True, 1), (300, 8, 1, 96, 96, False, 13), (700, 14, 2, 256, 128, False, 64),
    (3, 2, 1, 8, 6, False, 4), (4, 3, 3, 24, 2, True, 5), (2, 2, 2, 72, 0, False, 4)])
def test_append_rotary(gpu, T, H, G, D, rot, inter, P, dtype):
    dt = DT[dtype]
    g = torch.Generator(device="cuda").manual_seed(T + D)
    qkv = torch.randn(T, H + 2 * G, D, generator=g, device="cuda").to(dt)
    q, k, v = qkv[:, :H], qkv[:, H:H + G], qkv[:, H + G:]
    pages = -(-T // P) + 3
    kc = torch.randn(pages, P, G, D, generator=g, device="cuda").to(dt)
    vc = torch.randn(pages, P, G, D, generator=g, device="cuda").to(dt)
    k0, v0 = kc.clone(), vc.clone()
    slots = torch.randperm(pages * P, generator=g, device="cuda")[:T].contiguous()
    pos = torch.randint(0, 50, (T,), generator=g, device="cuda", dtype=torch.int32)
    cs = torch.randn(50, rot, generator=g, device="cuda")
    out = _C_ops.cache_append(k, v, kc, vc, slots, q=q, positions=pos, cos_sin=cs, interleaved=inter)
    close(out, *turned(q, cs, pos, inter), dt)
    wk, mk = turned(k, cs, pos, inter)
    close(kc.flatten(0, 1)[slots], wk, mk, dt)
    assert torch.equal(vc.flatten(0, 1)[slots], v)
    rest = torch.ones(pages * P, dtype=torch.bool, device="cuda")
    rest[slots] = False
    assert torch.equal(kc.flatten(0, 1)[rest], k0.flatten(0, 1)[rest])
    assert torch.equal(vc.flatten(0, 1)[rest], v0.flatten(0, 1)[rest])
    # in place, and the same bits
    q2 = q.clone()
    assert _C_ops.cache_append(k, v, kc, vc, slots, q=q2, positions=pos, cos_sin=cs, interleaved=inter, q_out=q2) is not None
    assert torch.equal(q2, out)


def test_append_without_rotary_and_skipped_tokens(gpu):
    T, G, D, P, pages = 9, 2, 64, 4, 5
    g = torch.Generator(device="cuda").manual_seed(3)
    k, v = (torch.randn(T, G, D, generator=g, device="cuda").half() for _ in range(2))
    kc, vc = (torch.zeros(pages, P, G, D, dtype=torch.float16, device="cuda") for _ in range(2))
    slots = torch.tensor([0, -1, 5, 20, 19, -7, 2 ** 40, 7, 8], device="cuda")
    assert _C_ops.cache_append(k, v, kc, vc, slots) is None
    keep = [0, 2, 4, 7, 8]
    want = torch.zeros_like(kc).flatten(0, 1)
    want[slots[keep]] = k[keep]
    assert torch.equal(kc.flatten(0, 1), want)
    # positions outside the table: nothing written, q is zero
    kc.zero_()
    pos = i32([0, 1, 2, 3, -1, 5, 6, 7, 4])
    q = torch.randn(T, 4, D, generator=g, device="cuda").half()
    out = _C_ops.cache_append(k, v, kc, vc, slots, q=q, positions=pos, cos_sin=torch.ones(5, D, device="cuda"))
    assert bool((out[[4, 5, 6, 7]] == 0).all()) and bool((out[[0, 1, 2, 3, 8]] != 0).any())
    assert sorted(kc.flatten(0, 1).abs().sum((1, 2)).nonzero().flatten().tolist()) == [0, 5, 8]


def test_append_odd_alignment_and_strides(gpu):
    # an odd element offset, and a cache whose keys and values share a buffer
    T, H, G, D, P, pages = 21, 4, 2, 64, 8, 6
    g = torch.Generator(device="cuda").manual_seed(4)
    flat = torch.randn(T * (H + 2 * G) * D + 1, generator=g, device="cuda").bfloat16()[1:]
    qkv = flat.view(T, H + 2 * G, D)
    q, k, v = qkv[:, :H], qkv[:, H:H + G], qkv[:, H + G:]
    kv = torch.zeros(pages, 2, P, G, D, dtype=torch.bfloat16, device="cuda")
    slots = torch.arange(T, device="cuda") + 3
    pos = torch.arange(T, device="cuda", dtype=torch.int32)
    cs = torch.randn(T, D, generator=g, device="cuda")
    out = _C_ops.cache_append(k, v, kv[:, 0], kv[:, 1], slots, q=q, positions=pos, cos_sin=cs)
    close(out, *turned(q, cs, pos, False), torch.bfloat16)
    close(kv[:, 0].flatten(0, 1)[slots], *turned(k, cs, pos, False), torch.bfloat16)
    assert torch.equal(kv[:, 1].flatten(0, 1)[slots], v)


# ------------------------------------------------------------ paged attention

def attend_reference(q, kc, vc, table, positions, rows, scale, window):
    """(out, bound) in 64 bits."""
    T, H, D = q.shape
    pages, P, G, _ = kc.shape
    dt = q.dtype
    out = torch.zeros(T, H, D, dtype=torch.float64)
    bound = torch.zeros(T, H, D, dtype=torch.float64)
    tab = table.cpu().tolist()
    for t in range(T):
        row = t if rows is None else int(rows[t])
        last = int(positions[t])
        if last < 0 or row < 0 or row >= len(tab):
            continue
        first = max(0, last + 1 - window) if window else 0
        j = [x for x in range(first, min(last + 1, len(tab[row]) * P)) if 0 <= tab[row][x // P] < pages]
        if not j:
            continue
        page = torch.tensor([tab[row][x // P] for x in j], device=kc.device)
        at = torch.tensor([x % P for x in j], device=kc.device)
        k, v = (c[page, at].double().cpu() for c in (kc, vc))  # [n, G, D]
        for h in range(H):
            g = h // (H // G)
            x = q[t, h].double().cpu()
            s = k[:, g] @ x * scale
            d = (D + 8) * 2.0 ** -24 * float((k[:, g].abs() @ x.abs()).max()) * abs(scale)
            p = torch.softmax(s, 0)
            out[t, h] = p @ v[:, g]
            bound[t, h] = U[dt] * 1.01 * out[t, h].abs() + TINY[dt] + (2 * d + 2.0 ** -15) * (p @ v[:, g].abs())
    return out, bound


def attend_case(lens, H, G, D, P, dt, seed=0, spare=3, width=None, sigma=2.0):
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
    q = (sigma * torch.randn(len(lens), H, D, generator=g, device="cuda")).to(dt)
    kc, vc = (torch.randn(pages, P, G, D, generator=g, device="cuda").to(dt) for _ in range(2))
    return q, kc, vc, table, i32([n - 1 for n in lens])


def attend_check(q, kc, vc, table, pos, rows=None, scale=None, window=0, out=None):
    got = _C_ops.paged_attention(q, kc, vc, table, pos, rows=rows, scale=scale, window=window, out=out)
    want, bound = attend_reference(q, kc, vc, table, pos, rows, q.shape[2] ** -0.5 if scale is None else scale, window)
    err = (got.double().cpu() - want).abs()
    assert bool((err <= bound).all()), (float((err - bound).max()), float(want.abs().max()))
    return got


LENS = [0, 1, 2, 31, 32, 33, 64, 127, 129, 300, 513]


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("H,G,D,P", [
    (4, 4, 128, 16), (8, 2, 128, 32), (8, 1, 64, 8), (6, 2, 80, 16), (7, 1, 96, 64), (4, 2, 256, 16), (16, 1, 128, 16),
    (17, 1, 64, 16), (40, 2, 128, 128), (3, 3, 8, 16), (4, 2, 72, 24), (2, 1, 112, 8), (4, 4, 128, 1), (8, 2, 64, 7),
    (5, 5, 248, 20), (16, 1, 256, 16), (32, 2, 200, 8)])
def test_attention_heads_and_pages(gpu, H, G, D, P, dtype):
    attend_check(*attend_case(LENS, H, G, D, P, DT[dtype]))


@pytest.mark.parametrize("window", [1, 7, 32, 100, 1000])
@pytest.mark.parametrize("P", [16, 5])
def test_attention_window(gpu, window, P):
    attend_check(*attend_case(LENS, 4, 2, 128, P, torch.float16), window=window)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("lens,H,G,D,P", [
    ([20000], 8, 2, 128, 64), ([5000, 1, 0, 9001], 4, 4, 64, 16),
    ([1, 7, 30000, 300, 2], 4, 1, 128, 32), ([40] * 70 + [25000] + [3] * 20, 8, 4, 64, 16), ([18000, 20000], 5, 1, 64, 8), ([3000] * 3, 32, 4, 80, 16), ([4097], 2, 1, 256, 128)])
def test_attention_long(gpu, lens, H, G, D, P, dtype):
    attend_check(*attend_case(lens, H, G, D, P, DT[dtype]))


def test_attention_many_short_requests(gpu):
    rng = np.random.default_rng(5)
    attend_check(*attend_case(rng.integers(0, 60, 400).tolist(), 4, 2, 64, 16, torch.bfloat16, width=40))


def test_attention_rows_of_one_request(gpu):
    # the tokens of a prompt (each its own position), padding, unknown rows
    q, kc, vc, table, _ = attend_case([70, 40, 90], 8, 2, 128, 16, torch.float16)
    rows = i32([1, 1, 1, 0, -1, 2, 2, 3, 0, 2 ** 31 - 1])
    pos = i32([37, 38, 39, 69, -1, 0, 88, 4, -1, 3])
    q = torch.randn(10, 8, 128, device="cuda").half()
    got = attend_check(q, kc, vc, table, pos, rows=rows)
    assert bool((got[[4, 7, 8, 9]] == 0).all())


def test_attention_hides_whatever_masked_places_hold(gpu):
    for P in (16, 24):
        q, kc, vc, table, pos = attend_case([5, 33, 100, 1], 4, 2, 128, P, torch.float16)
        want = attend_check(q, kc, vc, table, pos, window=30)
        seen = torch.zeros(kc.shape[0], P, dtype=torch.bool, device="cuda")
        for r, n in enumerate([5, 33, 100, 1]):
            for j in range(max(0, n - 30), n):
                seen[int(table[r, j // P]), j % P] = True
        for bad in (float("nan"), float("inf"), -65504.0):
            k2, v2 = kc.clone(), vc.clone()
            k2[~seen] = bad
            v2[~seen] = bad
            assert torch.equal(_C_ops.paged_attention(q, k2, v2, table, pos, window=30), want)


def test_attention_pages_outside_the_cache_are_not_seen(gpu):
    q, kc, vc, table, pos = attend_case([100, 100, 40], 4, 2, 64, 16, torch.bfloat16)
    table[0, 2] = -1
    table[0, 4] = kc.shape[0]
    table[1, :] = 2 ** 31 - 1  # sees nothing
    pos[2] = 5000              # past the table
    got = attend_check(q, kc, vc, table, pos)
    assert bool((got[1] == 0).all())


def test_attention_extreme_scores(gpu):
    q, kc, vc, table, pos = attend_case([3, 200, 64], 4, 2, 64, 16, torch.float16)
    attend_check(q, kc, vc, table, pos, scale=0.0)       # uniform weights
    attend_check(q * 30, kc, vc, table, pos, scale=1.0)  # one weight takes all
    attend_check(q, kc, vc, table, pos, scale=-0.125)
    # a key of infinite score in sight is NaN as in the formula; a hidden one is nothing
    kc[int(table[1, 3]), 2] = float("inf")
    out = _C_ops.paged_attention(q, kc, vc, table, pos)
    assert bool(out[1].isnan().any()) and not bool(out[[0, 2]].isnan().any())
    # scores ever growing: every key raises the running maximum
    n = 400
    q, kc, vc, table, pos = attend_case([n], 2, 1, 64, 16, torch.bfloat16)
    q.fill_(1.0)
    for j in range(n):
        kc[int(table[0, j // 16]), j % 16] = j / 8.0
    attend_check(q, kc, vc, table, pos, scale=0.05)
    # scores far below zero: exp of them alone would vanish
    attend_check(q, -kc - 60, vc, table, pos, scale=1.0)


def test_attention_strided_views(gpu):
    # queries out of a joined projection, the cache's keys and values side by
    # side, a table that is part of a wider one, an output in head order
    q, kc, vc, table, pos = attend_case(LENS, 6, 3, 64, 16, torch.float16)
    want = attend_check(q, kc, vc, table, pos)
    wide = torch.randn(len(LENS), 20, 64, device="cuda").half()
    wide[:, 3:9] = q
    kv = torch.stack([kc, vc], 1).contiguous()
    t2 = torch.zeros(len(LENS), table.shape[1] + 9, dtype=torch.int32, device="cuda")
    t2[:, :table.shape[1]] = table
    out = torch.empty(6, len(LENS), 64, dtype=torch.float16, device="cuda").transpose(0, 1)
    got = _C_ops.paged_attention(wide[:, 3:9], kv[:, 0], kv[:, 1], t2[:, :table.shape[1]], pos, out=out)
    assert got.data_ptr() == out.data_ptr() and torch.equal(got, want)
    # an odd element offset of q
    flat = torch.empty(q.numel() + 1, dtype=torch.float16, device="cuda")[1:].view(q.shape)
    flat.copy_(q)
    assert torch.equal(_C_ops.paged_attention(flat, kc, vc, table, pos), want)


def test_attention_past_32_bit_offsets(gpu):
    # a cache of 2^32 + elements, the request's pages at its end
    P, G, D = 16, 2, 128
    pages = (1 << 32) // (P * G * D) + 40
    cache = torch.empty(pages, P, G, D, dtype=torch.float16, device="cuda")
    cache[-40:].normal_()
    table = (pages - 1 - torch.arange(30, device="cuda", dtype=torch.int32))[None].contiguous()
    q = torch.randn(1, 4, D, device="cuda").half()
    got = _C_ops.paged_attention(q, cache, cache, table, i32([450]))
    small = (39 - torch.arange(30, device="cuda", dtype=torch.int32))[None].contiguous()
    assert torch.equal(got, attend_check(q, cache[-40:], cache[-40:], small, i32([450])))
    # and a slot written there
    k = torch.randn(1, G, D, device="cuda").half()
    _C_ops.cache_append(k, k, cache, cache, torch.tensor([pages * P - 3], device="cuda"))
    assert torch.equal(cache[-1, P - 3], k[0])


@pytest.mark.parametrize("P", [32, 28])
def test_attention_last_key_numbers(gpu, P):
    # windows at the end of the widest table there is (one page in every place)
    W = ((1 << 31) - 512) // P
    table = torch.zeros(1, W, dtype=torch.int32, device="cuda")
    kc, vc = (torch.randn(1, P, 1, 8, device="cuda").half() for _ in range(2))
    q = torch.randn(1, 2, 8, device="cuda").half()
    for back, window in ((1, 1), (1, 300), (40, 1000), (0, 70)):
        last = W * P - back  # (back 0: one key past the table, not seen)
        got = _C_ops.paged_attention(q, kc, vc, table, i32([last]), window=window)
        j = np.arange(max(0, last + 1 - window), min(last + 1, W * P)) % P
        s = (q[0].double() @ kc[0, :, 0].double().T.contiguous())[:, torch.tensor(j).cuda()] * 8 ** -0.5
        want = torch.softmax(s, -1) @ vc[0, :, 0].double()[torch.tensor(j).cuda()].contiguous()
        # FP16's rounding of values up to |v| <= 4, and FP32 sums behind it
        assert float((got[0].double() - want).abs().max()) <= 2 ** -9


def test_attention_is_the_same_every_time_and_on_other_streams(gpu):
    q, kc, vc, table, pos = attend_case([9000, 17, 4000], 8, 2, 128, 16, torch.bfloat16)
    want = attend_check(q, kc, vc, table, pos)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        assert torch.equal(_C_ops.paged_attention(q, kc, vc, table, pos), want)
        with torch.cuda.stream(s):
            got = _C_ops.paged_attention(q, kc, vc, table, pos)
        s.synchronize()
        assert torch.equal(got, want)


def test_step_append_attend_captured_and_replayed(gpu):
    """A serving step in a graph: replayed with other lengths and contents,
    each time the eager result."""
    P, W, H, G, D, T = 16, 40, 8, 2, 64, 6
    g = torch.Generator(device="cuda").manual_seed(8)
    lengths, new = i32([0, 5, 100, 37]), i32([3, 1, 1, 1])
    table = torch.zeros(4, W, dtype=torch.int32, device="cuda")
    free = torch.randperm(120, generator=g, device="cuda").to(torch.int32)
    pool = i32([0, 0])
    kc, vc = (torch.randn(120, P, G, D, generator=g, device="cuda").half() for _ in range(2))
    qkv = torch.randn(T, H + 2 * G, D, generator=g, device="cuda").half()
    cs = torch.randn(1000, D, generator=g, device="cuda")

    def step():
        L, p, _, rows, pos, slots = _C_ops.page_step(lengths, new, table, free, pool, P, T)
        q = _C_ops.cache_append(qkv[:, H:H + G], qkv[:, H + G:], kc, vc, slots, q=qkv[:, :H], positions=pos, cos_sin=cs)
        return _C_ops.paged_attention(q, kc, vc, table, pos, rows=rows), L, p

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
        out, L, p = step()
    for i in range(4):
        qkv.copy_(torch.randn(qkv.shape, generator=g, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in (out, L, p)]
        for a, b in zip(got, step()):
            assert torch.equal(a, b), i
        attend_check(*[torch.randn(2, 4, D, device="cuda").half(), kc, vc, table[:2].contiguous(), i32([4, 5])])
        new.copy_(i32([[1, 1, 1, 1], [0, 2, 0, 3], [2, 2, 1, 1], [6, 0, 0, 0]][i]))


# ------------------------------------------------------------------- refusals

def test_refusals(gpu):
    q, kc, vc, table, pos = attend_case([5, 9], 4, 2, 64, 16, torch.float16)
    A = _C_ops.paged_attention
    for args, msg in [
            ((q.cpu(), kc, vc, table, pos), "device"), ((q.float(), kc, vc, table, pos), "dtype"),
            ((q, kc, vc.bfloat16(), table, pos), "one dtype"), ((q, kc.float(), vc.float(), table, pos), "float16 or bfloat16"),
            ((q[:, :3], kc, vc, table, pos), "multiple of kv_heads"), ((q, kc, vc, table.long(), pos), "block_table"),
            ((q, kc, vc, table, pos.long()), "positions"), ((q, kc, vc, table[:1], pos), "rows of block_table"),
            ((q, kc, vc, table, pos[:1]), "positions"), ((q[..., :60], kc[..., :60], vc[..., :60], table, pos), "head_dim"),
            ((q, kc[..., ::2], vc[..., ::2], table, pos), "contiguous"), ((q, kc, vc[:1], table, pos), "kv_heads")]:
        with pytest.raises(RuntimeError, match=msg):
            A(*args)
    with pytest.raises(RuntimeError, match="window"):
        A(q, kc, vc, table, pos, window=-1)
    with pytest.raises(RuntimeError, match="out"):
        A(q, kc, vc, table, pos, out=q[:, :2])
    with pytest.raises(RuntimeError, match="overlap"):
        A(q, kc, vc, table, pos, out=q[:, :1].expand(2, 4, 64))
    odd = torch.zeros(kc.numel() + 8, dtype=kc.dtype, device="cuda")[1:1 + kc.numel()].view(kc.shape)
    with pytest.raises(RuntimeError, match="16-byte"):
        A(q, odd, vc, table, pos)
    k, slots = torch.zeros(2, 2, 64, dtype=torch.float16, device="cuda"), torch.zeros(2, dtype=torch.int64, device="cuda")
    cs = torch.zeros(4, 64, device="cuda")
    C = _C_ops.cache_append
    for args, kw, msg in [
            ((k, k, kc, vc, slots.int()), {}, "slots"), ((k[:, :1], k, kc, vc, slots), {}, "kv_heads"),
            ((k.bfloat16(), k, kc, vc, slots), {}, "dtype"), ((k, k, kc, vc, slots), {"q": q}, "cos_sin"),
            ((k, k, kc, vc, slots), {"cos_sin": cs}, "positions"),
            ((k, k, kc, vc, slots), {"cos_sin": cs[:, :63].contiguous(), "positions": pos}, "rot"),
            ((k, k, kc, vc, slots), {"cos_sin": cs.half(), "positions": pos}, "float32"),
            ((k, k, kc, vc, slots), {"q": q, "cos_sin": cs, "positions": pos, "q_out": q[:, :2]}, "q_out"),
            ((k, k, kc, vc, slots), {"q_out": q}, "q_out")]:
        with pytest.raises(RuntimeError, match=msg):
            C(*args, **kw)
    z = torch.zeros(2, dtype=torch.int32, device="cuda")
    S = _C_ops.page_step
    for args, msg in [((z, z[:1], table, z, z, 16, 2), "new_tokens"), ((z, z, table[:1], z, z, 16, 2), "block_table"),
                      ((z, z, table, z, z, 0, 2), "page_size"), ((z, z, table, z, z, 16, -1), "tokens"),
                      ((z.long(), z, table, z, z, 16, 2), "lengths"), ((z, z, table, z, z[:1], 16, 2), "pool"),
                      ((z, z, table, z.float(), z, 16, 2), "free_pages")]:
        with pytest.raises(RuntimeError, match=msg):
            S(*args)


def test_ctypes_binding_gives_the_same(gpu, monkeypatch):
    q, kc, vc, table, pos = attend_case(LENS, 4, 2, 64, 16, torch.float16)
    want = _C_ops.paged_attention(q, kc, vc, table, pos, window=50)
    k = torch.randn(len(LENS), 2, 64, device="cuda").half()
    slots = torch.arange(len(LENS), device="cuda")
    cs = torch.randn(600, 64, device="cuda")
    step = (i32([3, 5]), i32([2, 1]), torch.zeros(2, 4, dtype=torch.int32, device="cuda"), i32([3, 4, 5]), i32([0, 0]), 4, 5)
    a = [_C_ops.cache_append(k, k, kc.clone(), vc.clone(), slots, q=q, positions=pos, cos_sin=cs), *_C_ops.page_step(*step)]
    monkeypatch.setattr(_lib, "torch_ops", lambda: None)
    assert torch.equal(_C_ops.paged_attention(q, kc, vc, table, pos, window=50), want)
    b = [_C_ops.cache_append(k, k, kc.clone(), vc.clone(), slots, q=q, positions=pos, cos_sin=cs), *_C_ops.page_step(*step)]
    for x, y in zip(a, b):
        assert torch.equal(x, y)
    test_refusals(gpu)
