"""Rotary positions, the paged cache, attention over it and eviction, against plain implementations in 64 bits.

Tolerances are sums of roundings; where one is used its terms stand beside it.  u = 2^-24 is half a step of fp32.
"""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0**-24
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}
HALF_STEP = {"f16": (2.0**-11, 2.0**-25), "bf16": (2.0**-8, 2.0**-134), "e4m3": (2.0**-4, 2.0**-10)}  # of a value, and at least
LARGEST = {"f16": 65504.0, "bf16": 3.3895313892515355e38, "e4m3": 448.0}


@pytest.fixture(scope="module")
def capi(native_lib, cuda_device):
    native_lib.device_fault(clear=True)
    return native_lib


@pytest.fixture(autouse=True)
def no_fault(capi):
    yield
    assert capi.device_fault(clear=True) == 0


def generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def randn(g, *shape, dtype=torch.float32):
    if dtype == torch.float8_e4m3fn:
        return (torch.randn(shape, generator=g, device="cuda") * 8).to(dtype)
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def pool(g, pages, slots, heads, dim, dtype, layout="slots"):
    """Two tensors [pages, slot, head, element]; "heads": heads ahead of slots in memory, "both": keys and values of a page side by side."""
    if layout == "both":
        t = randn(g, pages, 2, slots, heads, dim, dtype=dtype)
        return t[:, 0], t[:, 1]
    shape = (pages, heads, slots, dim) if layout == "heads" else (pages, slots, heads, dim)
    both = [randn(g, *shape, dtype=dtype) for _ in range(2)]
    return [t.transpose(1, 2) for t in both] if layout == "heads" else both


def table_for(g, lengths, page, spare=2, extra=0):
    """A page table for these lengths over distinct pages in random order, -1 behind; and how many pages the pool has."""
    need = [-(-n // page) for n in lengths]
    total = sum(need) + spare
    order = torch.randperm(total, generator=g, device="cuda").tolist()
    rows, at = [], 0
    for n in need:
        rows.append(order[at:at + n] + [-1] * (max(need + [1]) + extra - n))
        at += n
    return i32(rows), total


# ---- rotary positions ------------------------------------------------------------------------------------------------
def rotated(x, positions, radians, mscale, interleaved):
    """[T, H, D] in 64 bits -> (turned, the bound's a, b size)."""
    x, r = x.double(), 2 * len(radians)
    angle = positions.double().cpu()[:, None] * torch.tensor(radians, dtype=torch.float64)
    # a position times a frequency in double precision is off by 2^-53 of some 10^9 turns at most: 1e-7; the library's is exact, so the
    # reference's own product is what far positions are compared up to
    cos, sin = (f(angle).to(x.device)[:, None, :] * mscale for f in (torch.cos, torch.sin))
    y, size = x.clone(), x.abs()
    a, b = (x[..., 0:r:2], x[..., 1:r:2]) if interleaved else (x[..., : r // 2], x[..., r // 2:r])
    pair = [(a * cos - b * sin), (b * cos + a * sin)]
    at = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2), slice(r // 2, r))
    for k in range(2):
        y[..., at[k]] = pair[k]
        size[..., at[k]] = (a.abs() + b.abs()) * mscale
    return y, size


def rope_bound(size, positions):
    # half turns to half a bit of 1: pi 2^-25 = 1.6 u in the angle; sincospif to 2 ulp = 4 u; times mscale, u; products and sum 3 u:
    # under 10 u of |a| + |b|.  The reference's angle: position * frequency to 2^-53.
    return size * (10 * U + positions.double().abs()[:, None, None].to(size.device) * 2.0**-52)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("T,H,D,R", [(1, 1, 2, 2), (1, 32, 128, 128), (3, 5, 80, 20), (7, 3, 96, 48), (2, 7, 64, 6), (33, 25, 80, 20), (5, 2, 256, 256),
                                     (2, 3, 62, 30), (700, 9, 128, 64), (3000, 4, 64, 64), (2, 1, 1024, 1024), (1, 129, 16, 16)])
def test_rope(capi, T, H, D, R, interleaved):
    g = generator(T * H * D + R + interleaved)
    x = randn(g, T, H, D)
    positions = torch.randint(0, 100000, (T,), generator=g, device="cuda", dtype=torch.int32)
    radians = [10000.0 ** (-2.0 * i / R) for i in range(R // 2)]
    table, mscale = capi.rope_table(R, 10000.0, device="cuda")
    got = capi.rope(x, positions, table, interleaved=interleaved, mscale=mscale)
    want, size = rotated(x, positions, radians, 1.0, interleaved)
    assert ((got.double() - want).abs() <= rope_bound(size, positions)).all()
    assert torch.equal(got[..., R:], x[..., R:])
    same = x.clone()
    assert capi.rope(same, positions, table, interleaved=interleaved, out=same) is same and torch.equal(same, got)


@pytest.mark.parametrize("interleaved", [False, True])
def test_rope_positions_at_the_ends(capi, interleaved):
    """The first, the last and negative ones; a position's angle is exact however far."""
    g = generator(3)
    where = [0, 1, -1, 2**24, 2**24 + 1, 2**31 - 1, -2**31, 10**9]
    x, positions = randn(g, len(where), 3, 64), i32(where)
    radians = [math.pi * 2.0 ** -(i + 1) for i in range(32)]  # whole fractions of a turn: the angle is a residue, exact in integers
    table, _ = capi.rope_table(64, frequencies=radians, device="cuda")
    got = capi.rope(x, positions, table, interleaved=interleaved).double()
    # 2 pi / 2^(i + 2): the angle is 2 pi (p mod 2^(i + 2)) / 2^(i + 2); the table's entry is off by 2^-53 of itself (the double's pi)
    left = torch.tensor([[(p % 2 ** (i + 2)) for i in range(32)] for p in where], dtype=torch.float64)
    residue = left / torch.tensor([2.0 ** (i + 2) for i in range(32)], dtype=torch.float64)
    cos, sin = (f(2 * math.pi * residue)[:, None, :].cuda() for f in (torch.cos, torch.sin))
    at = (slice(0, 64, 2), slice(1, 64, 2)) if interleaved else (slice(0, 32), slice(32, 64))
    a, b = x[..., at[0]].double(), x[..., at[1]].double()
    size = a.abs() + b.abs()
    bound = size * (10 * U + torch.tensor(where, dtype=torch.float64).abs()[:, None, None].cuda() * 4 * 2.0**-53)
    assert ((got[..., at[0]] - (a * cos - b * sin)).abs() <= bound).all()
    assert ((got[..., at[1]] - (b * cos + a * sin)).abs() <= bound).all()


def test_rope_strides_and_alignment(capi):
    """Rows and heads of a wider tensor, beginning at any float; what lies between is left alone."""
    g = generator(4)
    table, mscale = capi.rope_table(32, 10000.0, "yarn", 8.0, 512, device="cuda")
    positions = i32([5, 0, 70000])
    wide = randn(g, 3, 4, 100)
    dense = capi.rope(wide[:, 1:3, 3:67].contiguous(), positions, table, mscale=mscale)
    out = torch.full((3, 5, 90), 7.0, device="cuda")
    capi.rope(wide[:, 1:3, 3:67], positions, table, mscale=mscale, out=out[:, 1:3, 5:69])
    assert torch.equal(out[:, 1:3, 5:69], dense)
    out[:, 1:3, 5:69] = 7.0
    assert (out == 7.0).all()
    row = randn(g, 1, 2, 64).expand(3, 2, 64)  # one row for all positions
    assert torch.equal(capi.rope(row, positions, table), capi.rope(row.contiguous(), positions, table))


def test_rope_sines_of_exact_angles(capi):
    """Pairs (1, 0): what comes out are cosine and sine themselves, of angles that are exact in integers."""
    n = 1 << 16
    g = generator(46)
    steps = torch.randint(-2**63, 2**63 - 1, (8,), generator=g, device="cuda", dtype=torch.int64)
    positions = torch.randint(0, 2**24, (n,), generator=g, device="cuda", dtype=torch.int32)
    x = torch.zeros((n, 1, 16), device="cuda")
    x[..., :8] = 1.0
    got = capi.rope(x, positions, steps).double()[:, 0]
    angle = positions.long()[:, None] * steps  # modulo 2^64, a turn
    # the angle in 64 bits: its upper 53 bits, to 2^-52 of a turn
    radians = (angle >> 11).double() * (2 * math.pi / 2.0**53)
    for part, f in ((got[:, :8], torch.cos), (got[:, 8:], torch.sin)):
        # what is left of the angle: 2^-27 and 2^-33 half turns, pi of which 0.4 u; sincospif to 2 ulp, which for values up to 1 is 2 u; the products with 1 and 0 are exact
        assert ((part - f(radians)).abs() <= 2.5 * U).all()


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("T,H,D,R,shift", [(3, 2, 1024, 1024, 1), (2, 3, 1024, 1022, 0), (2, 1, 1022, 1022, 3), (5, 2, 1022, 6, 2), (3, 2, 514, 514, 1),
                                           (700, 3, 514, 258, 0), (1, 2, 1022, 1020, 2), (2, 2, 516, 512, 1)])
def test_rope_wide_heads_of_any_alignment(capi, T, H, D, R, shift, interleaved):
    """Heads with more pairs than a block has threads: taken pair by pair where they begin at any float, or do not divide by four."""
    g = generator(D + R + shift)
    wide = randn(g, T, H, D + 5)
    x = wide[..., shift:shift + D]
    positions = torch.randint(0, 100000, (T,), generator=g, device="cuda", dtype=torch.int32)
    table, mscale = capi.rope_table(R, 10000.0, device="cuda")
    want, size = rotated(x, positions, [10000.0 ** (-2.0 * i / R) for i in range(R // 2)], 1.0, interleaved)
    got = capi.rope(x, positions, table, interleaved=interleaved, mscale=mscale)
    assert ((got.double() - want).abs() <= rope_bound(size, positions)).all()
    assert torch.equal(got[..., R:], x[..., R:])
    before = wide.clone()
    capi.rope(x, positions, table, interleaved=interleaved, mscale=mscale, out=x)  # where it lies
    assert torch.equal(x, got)
    before[..., shift:shift + D] = got
    assert torch.equal(wide, before)


def test_rope_refuses_what_does_not_fit(capi):
    table, _ = capi.rope_table(64, device="cuda")
    x = torch.zeros((2, 3, 32), device="cuda")
    with pytest.raises(capi.JqError) as e:
        capi.rope(x, i32([0, 1]), table)
    assert e.value.status == capi.ERR_SHAPE
    with pytest.raises(ValueError):
        capi.rope(x, torch.tensor([0, 1], dtype=torch.int32), table)  # on the host
    assert capi.rope(torch.zeros((0, 3, 64), device="cuda"), i32([]), table).shape == (0, 3, 64)


# ---- into the cache ----------------------------------------------------------------------------------------------------
def within_a_rounding(got, want, error, kind, scale=1.0):
    """Stored elements against a value known up to `error`: half a step of the value, and the error."""
    rel, least = HALF_STEP[kind]
    w = (want / scale).clamp(-LARGEST[kind], LARGEST[kind])
    e = error / scale
    return ((got.double() - w).abs() <= (w.abs() + e) * rel * (1 + 4 * U) + least + e + w.abs() * U).all()


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("Hq,Hk,D,R,page,layout,interleaved", [
    (32, 8, 128, 128, 16, "slots", False), (4, 4, 64, 64, 1, "heads", True), (7, 1, 80, 20, 24, "slots", True), (3, 3, 96, 48, 5, "both", False),
    (16, 2, 256, 256, 128, "heads", False), (0, 2, 16, 16, 3, "slots", False), (5, 5, 48, 6, 7, "both", True), (2, 2, 112, 2, 64, "slots", False)])
@pytest.mark.parametrize("T", [1, 6, 700])
def test_rope_append(capi, kind, Hq, Hk, D, R, page, layout, interleaved, T):
    g = generator(Hq + 10 * Hk + D + R + T)
    lengths = [13, 0, 200 + page, 1]
    k_scale, v_scale = (0.25, 0.125) if kind == "e4m3" else (1.0, 1.0)
    table, mscale = capi.rope_table(R, 500.0, "yarn", 4.0, 64, device="cuda")
    # rows in any order among the sequences, each behind what its sequence holds
    seqs = torch.randint(0, 4, (T,), generator=g, device="cuda").tolist()
    filled, index = list(lengths), []
    for s in seqs:
        index.append(filled[s])
        filled[s] += 1
    pages, total = table_for(g, filled, page)
    k, v = pool(g, total, page, Hk, D, TYPES[kind], layout)
    k0, v0 = k.clone(), v.clone()
    qkv = randn(g, T, (Hq + 2 * Hk) * D)
    positions = torch.randint(0, 9000, (T,), generator=g, device="cuda", dtype=torch.int32)
    q = capi.rope_append(qkv, positions, table, k, v, pages, i32(index), seqs=i32(seqs), interleaved=interleaved, mscale=mscale, k_scale=k_scale,
                         v_scale=v_scale)
    x = qkv.view(T, Hq + 2 * Hk, D)
    plain = capi.rope(x[:, :Hq], positions, table, interleaved=interleaved, mscale=mscale)
    assert torch.equal(q, plain)  # (checked above)
    turned = capi.rope(x[:, Hq:Hq + Hk], positions, table, interleaved=interleaved, mscale=mscale).double()
    at = torch.tensor(index, device="cuda")
    where = pages[torch.tensor(seqs, device="cuda"), at // page].long(), at % page
    # the kernel's own fp32 rotation rounds as rope()'s does, give or take a contraction: 2 u of |a| + |b| <= 2 max |x|
    assert within_a_rounding(k[where].float(), turned, 4 * U * x.abs().max().item() * mscale, kind, k_scale)
    assert within_a_rounding(v[where].float(), x[:, Hq + Hk:].double(), 0.0, kind, v_scale)
    # nothing else was touched
    k[where], v[where] = k0[where], v0[where]
    assert torch.equal(k.contiguous().view(torch.uint8), k0.contiguous().view(torch.uint8))
    assert torch.equal(v.contiguous().view(torch.uint8), v0.contiguous().view(torch.uint8))


def test_rope_append_padding_and_bad_pages(capi):
    """Rows of no sequence or index leave the cache alone, and so does a page that does not exist, which is reported."""
    g = generator(8)
    table, _ = capi.rope_table(64, device="cuda")
    k, v = pool(g, 6, 16, 2, 64, torch.float16)
    k0, v0 = k.clone(), v.clone()
    pages = i32([[0, 1], [2, -1], [6, 3]])
    qkv = randn(g, 7, 8 * 64)
    positions = i32(list(range(7)))

    def call(index, seqs):
        return capi.rope_append(qkv, positions, table, k, v, pages, i32(index), seqs=i32(seqs))

    q = call([0, -1, 32, 5, 2**31 - 1, 1, -2**31], [-1, 0, 1, 3, 0, 2**31 - 1, 2])
    assert torch.equal(k, k0) and torch.equal(v, v0) and capi.device_fault() == 0
    assert torch.equal(q, capi.rope(qkv.view(7, 8, 64)[:, :4], positions, table))
    call([16, 0, 17, 3, 18, 4, 0], [1, 2, 1, 2, 1, 2, -1])  # pages -1 and 6
    assert torch.equal(k, k0) and torch.equal(v, v0)
    assert capi.device_fault(clear=False) == capi.FAULT_BAD_PAGE and capi.device_fault(clear=True) == capi.FAULT_BAD_PAGE
    call([15] + [0] * 6, [0] + [-1] * 6)  # and the next call is right
    assert capi.device_fault() == 0 and not torch.equal(k[0, 15], k0[0, 15])
    assert torch.equal(v[0, 15], qkv.view(7, 8, 64)[0, 6:].half())


@pytest.mark.parametrize("page_first", [False, True])
def test_a_bad_page_hides_no_wait_that_gave_up(capi, page_first):
    """Whichever came first: the wait, whose results are not valid, is reported, then the page; neither is lost when the other is cleared."""
    table, _ = capi.rope_table(16, device="cuda")
    k, v = pool(generator(2), 1, 1, 1, 16, torch.float16)
    flags, epoch = torch.zeros(64, dtype=torch.int32, device="cuda"), i32([1])

    def bad_page():
        capi.rope_append(torch.zeros((1, 32), device="cuda"), i32([0]), table, k, v, i32([[1]]), i32([0]))
        torch.cuda.synchronize()

    def wait_for_nothing():  # bands that no rank sends: 4096 looks, then the kernel returns
        capi.set_option(capi.OPT_WAIT_POLL_LIMIT, 4096)
        try:
            capi.allgather_wait(flags.device, flags.data_ptr(), 1, epoch)
            torch.cuda.synchronize()
        finally:
            capi.set_option(capi.OPT_WAIT_POLL_LIMIT, 0)

    for report in (bad_page, wait_for_nothing) if page_first else (wait_for_nothing, bad_page):
        report()
    code = capi.ctypes.c_int(0)
    read = lambda clear: (capi.lib().jq_device_fault(clear, capi.ctypes.byref(code)), code.value)  # noqa: E731
    assert read(0) == (capi.ERR_TIMEOUT, 2)
    assert read(1) == (capi.ERR_TIMEOUT, 2)
    assert read(0) == (capi.ERR_INVALID_ARG, capi.FAULT_BAD_PAGE)
    assert read(1) == (capi.ERR_INVALID_ARG, capi.FAULT_BAD_PAGE)
    assert read(1) == (capi.OK, 0)


@pytest.mark.parametrize("kind", list(TYPES))
def test_rope_append_values_beyond_the_type(capi, kind):
    table, _ = capi.rope_table(16, device="cuda")
    k, v = pool(generator(1), 1, 1, 1, 16, TYPES[kind])
    big = [1e38, -1e38, math.inf, -math.inf, math.nan, 3.4e38, -3.4e38, 448.0, 464.0, 480.0, 65504.0, 65519.0, 65520.0, 1e-30, 0.0, -0.0]
    qkv = torch.tensor([0.0] * 16 + big, device="cuda")[None]
    capi.rope_append(qkv, i32([0]), table, k, v, i32([[0]]), i32([0]))
    got = v[0, 0, 0].float().tolist()
    for x, y in zip(big, got):
        if math.isnan(x):
            assert math.isnan(y)
        else:
            want = max(-LARGEST[kind], min(LARGEST[kind], x))
            assert abs(y) <= LARGEST[kind] and abs(y - want) <= abs(want) * HALF_STEP[kind][0] + HALF_STEP[kind][1], (x, y)


def test_rope_append_in_place_and_from_a_wider_row(capi):
    g = generator(9)
    table, _ = capi.rope_table(64, device="cuda")
    pages, positions, index = i32([[0], [1]]), i32([3, 4]), i32([2, 7])
    wide = randn(g, 2, 6 * 64 + 40)
    qkv = wide[:, 8:8 + 6 * 64]
    k, v = pool(g, 2, 8, 1, 64, torch.bfloat16)
    k2, v2 = k.clone(), v.clone()
    q = capi.rope_append(qkv.contiguous(), positions, table, k, v, pages, index)
    edges = wide.clone()
    where = qkv.view(2, 6, 64) if qkv.is_contiguous() else qkv.unflatten(1, (6, 64))
    capi.rope_append(qkv, positions, table, k2, v2, pages, index, q_out=where[:, :4])
    assert torch.equal(where[:, :4], q) and torch.equal(k, k2) and torch.equal(v, v2)
    wide[:, 8:8 + 4 * 64] = edges[:, 8:8 + 4 * 64]
    assert torch.equal(wide, edges)


# ---- attention ---------------------------------------------------------------------------------------------------------
def attended(q, k, v, pages, lens, page, scale, window=0, seqs=None, k_scale=1.0, v_scale=1.0):
    """In 64 bits -> (out [T, H, D], weights per row and key head as lists, bound on the difference, bound on a share's relative error)."""
    T, H, D = q.shape
    Hk = k.shape[2]
    G = H // Hk
    out, shares, far = torch.zeros((T, H, D), dtype=torch.float64, device="cuda"), [], torch.zeros((T, H, 1), dtype=torch.float64, device="cuda")
    worst = 0.0
    for t in range(T):
        s = t if seqs is None else seqs[t]
        shares.append([])
        if s < 0:
            continue
        n = min(max(lens[t], 0), pages.shape[1] * page)
        lo = max(0, n - window) if window else 0
        at = torch.arange(lo, n, device="cuda")
        where = pages[s, at // page].long()
        fine = (where >= 0) & (where < k.shape[0])
        where, slot = where[fine], at[fine] % page
        for h in range(Hk):
            if not len(where):
                shares[t].append((at[fine], torch.zeros(0, device="cuda").double()))
                continue
            kk, vv = k[where, slot, h].double() * k_scale, v[where, slot, h].double() * v_scale
            qq = q[t, h * G:(h + 1) * G].double()
            p = torch.softmax(qq @ kk.T * scale, -1)
            out[t, h * G:(h + 1) * G] = p @ vv
            shares[t].append((at[fine], p.sum(0)))
            # A logit's products sum up to S = scale |q| . |k|.  The query's parts leave 4 u of its largest element (22 bits, taken for every
            # element: 4 u max|q| sum|k|); the tensor cores drop less than 2 u of a partial sum per step, D / 16 steps of up to three parts, and
            # two more roundings: (3 D / 16 + 2) 2 u S.  Scaling, 2^x to 4 u and the subtraction of the maximum: (8 + |s|) u.
            size = (qq.abs() @ kk.abs().T * abs(scale)).max().item()
            widest = (qq.abs().amax() * kk.abs().sum(-1).max() * abs(scale)).item()
            d = (4 * widest + (3 * D / 16 + 2) * 2 * size + 8 + size) * U
            # shares carry d each way; values: six parts of two units, at 2 u, their sums over steps, warps and blocks (a hundred at most, u each,
            # for the sums are rounded)
            far[t, h * G:(h + 1) * G] = (2 * d + 120 * U) * vv.abs().max()
            worst = max(worst, 2 * d + 60 * U)
    return out, shares, far, worst


def check_attention(capi, g, kind, Hq, Hk, D, page, lens, layout="slots", window=0, seqs=None, table_seqs=None, poison=True, scale=None, q_size=1.5, weights=False,
                    negative=False):
    held = lens if table_seqs is None else table_seqs
    pages, total = table_for(g, [max(n, 0) for n in held], page, extra=1)
    k, v = pool(g, total, page, Hk, D, TYPES[kind], layout)
    k_scale, v_scale = (0.125, 0.25) if kind == "e4m3" else (1.0, 1.0)
    if poison:  # whatever no row may see is not a number
        seen = torch.zeros((total, page), dtype=torch.bool, device="cuda")
        for t, n in enumerate(lens):
            s = t if seqs is None else seqs[t]
            if s >= 0 and n > 0:
                at = torch.arange(max(0, n - window) if window else 0, n, device="cuda")
                seen[pages[s, at // page].long(), at % page] = True
        bad = torch.full((), math.nan, device="cuda").to(TYPES[kind])
        for t in (k, v):
            t.copy_(torch.where(seen[:, :, None, None], t.float(), bad.float()).to(TYPES[kind]))
    T = len(lens)
    q = randn(g, T, Hq, D) * q_size
    scale = (-1 if negative else 1) * (D**-0.5 if scale is None else scale)
    out = torch.full((T, Hq, D), 99.0, device="cuda")
    want_q8 = D % 32 == 0 and Hq * D % 128 == 0
    sums = torch.rand((T, Hk, pages.shape[1] * page), generator=g, device="cuda") if weights else None
    before = sums.clone() if weights else None
    xq = capi.paged_attention_q8_1(q, k, v, pages, i32(lens), seqs=None if seqs is None else i32(seqs), scale=scale, window=window, k_scale=k_scale,
                                   v_scale=v_scale, out=out, want_q8=want_q8, weights=sums)
    want, shares, far, worst = attended(q, k, v, pages, lens, page, scale, window, seqs, k_scale, v_scale)
    rows = [t for t in range(T) if seqs is None or seqs[t] >= 0]
    assert torch.isfinite(out).all()
    error = (out.double() - want).abs()
    assert (error[rows] <= far[rows]).all(), (error[rows] / far[rows].clamp(min=1e-300)).max()
    for t in range(T):
        if t not in rows:
            assert (out[t] == 99.0).all()
    if want_q8 and len(rows) == T:
        assert torch.equal(xq, capi.quantize_q8_1(out.view(T, Hq * D), capi.ORDER_COL_KSUPER, capi.S_D_SUM_Q))
    if weights:
        for t in range(T):
            for h in range(Hk):
                at, share = shares[t][h]
                rest = torch.ones(sums.shape[2], dtype=torch.bool, device="cuda")
                rest[at] = False
                assert torch.equal(sums[t, h][rest], before[t, h][rest])
                expect = before[t, h][at].double() + share
                assert ((sums[t, h][at].double() - expect).abs() <= share * worst + expect * 2 * U + 2.0**-120).all()
    return q, k, v, pages, out


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("Hq,Hk,D", [(1, 1, 16), (4, 4, 64), (8, 2, 128), (7, 1, 80), (24, 3, 96), (32, 2, 128), (16, 1, 64), (20, 1, 48), (3, 3, 256),
                                     (18, 2, 192), (48, 3, 112), (40, 1, 128)])
def test_attention_heads_and_sizes(capi, kind, Hq, Hk, D):
    check_attention(capi, generator(Hq + Hk * 50 + D), kind, Hq, Hk, D, 16, [1, 15, 16, 17, 0, 33, 100, 257])


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("page,layout", [(1, "slots"), (1, "heads"), (3, "both"), (16, "heads"), (24, "slots"), (32, "both"), (48, "heads"), (100, "slots"),
                                         (256, "both")])
def test_attention_pages_and_strides(capi, kind, page, layout):
    check_attention(capi, generator(page), kind, 8, 2, 64, page, [70, 1, 300, 2, 511], layout)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("D", [32, 144, 160, 176, 208, 224, 240])
def test_attention_heads_between_the_instances(capi, kind, D):
    """Widths that fill their instance's tiles in part."""
    check_attention(capi, generator(D), kind, 4, 2, D, 16, [1, 40, 333])
    check_attention(capi, generator(D), kind, 24, 2, D, 5, [1, 40, 333], weights=True)


@pytest.mark.parametrize("window", [0, 20])
def test_attention_lengths_beyond_the_table(capi, window):
    """They count as what the row of the table has room for; negative ones as nothing."""
    g = generator(48)
    k, v = pool(g, 4, 16, 2, 64, torch.float16)
    pages, q = i32([[3, 0], [1, 2], [0, 1]]), randn(g, 3, 4, 64)
    cut, beyond = torch.empty_like(q), torch.empty_like(q)
    capi.paged_attention_q8_1(q, k, v, pages, i32([32, 32, 0]), window=window, out=cut, want_q8=False)
    capi.paged_attention_q8_1(q, k, v, pages, i32([33, 2**31 - 1, -2**31]), window=window, out=beyond, want_q8=False)
    assert torch.equal(cut, beyond) and (beyond[2] == 0).all()


@pytest.mark.parametrize("rows,length,Hq,Hk", [(1, 1, 4, 4), (1, 40, 4, 1), (1, 3000, 8, 1), (1, 20011, 4, 2), (3, 5000, 8, 8), (40, 90, 8, 8), (200, 33, 4, 4),
                                               (33, 700, 16, 16), (600, 5, 2, 1), (5, 9000, 32, 2)])
@pytest.mark.parametrize("kind", ["f16", "bf16", "e4m3"])
def test_attention_divides_its_work(capi, kind, rows, length, Hq, Hk):
    """From one unit for the whole device to rows that end anywhere in a warp's or a block's stretch."""
    rng = np.random.default_rng(rows + length)
    lens = [length] + [int(n) for n in rng.integers(0, length + 1, rows - 1)]
    check_attention(capi, generator(rows * length), kind, Hq, Hk, 128, 16, lens, poison=rows * length < 60000)


@pytest.mark.parametrize("window", [1, 2, 15, 16, 17, 100, 1000])
@pytest.mark.parametrize("page", [16, 5])
def test_attention_window(capi, window, page):
    check_attention(capi, generator(window), "f16", 8, 2, 64, page, [1, 0, 16, 17, 99, 100, 101, 640, 641], window=window)
    check_attention(capi, generator(window), "bf16", 2, 1, 128, page, [2000], window=window, weights=True)


@pytest.mark.parametrize("kind", list(TYPES))
def test_attention_rows_of_the_same_sequence(capi, kind):
    """A prompt's tokens, drafted tokens, and padding: each row has its sequence and its length; rows of none are left as they were."""
    seqs = [2, 2, 2, 0, -1, 1, 1, -7, 3, 2]
    lens = [1, 2, 3, 200, 50, 0, 64, 9, 17, 130]
    check_attention(capi, generator(5), kind, 8, 4, 64, 16, lens, seqs=seqs, table_seqs=[200, 64, 130, 17])


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("scale,q_size,negative", [(1.0, 1e-20, False), (1e-3, 1e6, False), (0.1, 1.0, True), (0.0, 1.0, False), (2.0, 8.0, False), (1e-30, 1e30, False)])
def test_attention_scales(capi, kind, scale, q_size, negative):
    """Queries of any size, a scale that is negative or nothing, logits so far apart that one key takes all."""
    check_attention(capi, generator(6), kind, 4, 2, 64, 16, [33, 300], scale=scale, q_size=q_size, negative=negative)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("size", [1e4, 1e7, 1e8, 1e9, 1e12, 1e20, 1e30])
@pytest.mark.parametrize("tokens", [20, 300, 5000])
def test_attention_logits_of_any_size(capi, kind, size, tokens):
    """One key that is far ahead of the others: it is given all, however large its logit (a bit of which may be a thousand)."""
    g = generator(43)
    Hk, G, D, need = 2, 3, 64, -(-tokens // 16)
    k, v = pool(g, need, 16, Hk, D, TYPES[kind])
    k.copy_((torch.rand(k.shape, generator=g, device="cuda") / 4).to(TYPES[kind]))
    q = randn(g, 2, Hk * G, D)
    q += q.sign() * 0.5
    at = [3, 17, tokens - 1]
    pages = torch.arange(need, dtype=torch.int32, device="cuda").repeat(2, 1)
    # q . sign(q) * 2 = 2 |q|: 160 or so; of another head 2 q . sign(q'): 40 at most; of the rest |q| / 4
    q[1] = q[0]
    for h in range(Hk):
        for i in range(G):
            k[at[i] // 16, at[i] % 16, h] = (2 * q[0, h * G + i].sign()).to(TYPES[kind])
    q *= size
    weights, out = torch.zeros((2, Hk, need * 16), device="cuda"), torch.empty_like(q)
    scale = D**-0.5
    for w in (None, weights):
        capi.paged_attention_q8_1(q, k, v, pages, i32([tokens, tokens]), scale=scale, k_scale=0.125, v_scale=0.25, out=out, want_q8=False, weights=w)
        for h in range(Hk):
            for i in range(G):
                want = v[at[i] // 16, at[i] % 16, h].double() * 0.25
                # p = 1 in parts of 22 bits, 4 u; a step's products 2 u; sums over steps, warps and blocks with zeros; 1 / l, its factor and the product
                assert ((out[:, h * G + i].double() - want).abs() <= 20 * U * want.abs()).all(), (h, i)
    gained = torch.zeros_like(weights).double()
    for i in range(G):
        gained[:, :, at[i]] += 1
    assert ((weights.double() - gained).abs() <= 20 * U * gained).all()


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("n,below", [(64, 20.25), (1 << 16, 30.25), (1 << 16, 35.5), (1 << 12, 37.5), (1 << 16, 38.5), (1 << 12, 39.5), (1 << 12, 44.0)])
def test_attention_keys_that_have_next_to_nothing(capi, kind, n, below):
    """Of every 32 keys one has nearly all, and a value of nothing; the others have 2^-below of it each, and what is left is theirs."""
    D, page = 16, 64
    k, v = (torch.zeros((n // page, page, 1, D), device="cuda") for _ in range(2))
    k[:, ::32, 0, 0], v[:] = 1.0, 1.0
    v[:, ::32] = 0.0
    q = torch.zeros((1, 1, D), device="cuda")
    q[0, 0, 0] = logit = float(torch.tensor(below * math.log(2)))
    out = torch.empty_like(q)
    capi.paged_attention_q8_1(q, k.to(TYPES[kind]), v.to(TYPES[kind]), torch.arange(n // page, dtype=torch.int32, device="cuda")[None], i32([n]), scale=1.0, out=out,
                              want_q8=False)
    each = math.exp(-logit)
    want = 31 * each / (1 + 31 * each)
    # a share's relative error (see attended(); products of one element: size and widest are the logit); with fp16 parts, the rounding to 2^-40
    d = (4 * logit + (3 * D / 16 + 2) * 2 * logit + 8 + logit) * U
    assert ((out.double() - want).abs() <= want * (2 * d + 120 * U) + (0 if kind == "bf16" else 31 * 2.0**-40)).all(), (out[0, 0, 0].item(), want)


@pytest.mark.parametrize("key,scale", [(1e38, 0.0), (1e30, 0.0), (3e38, 1e-43), (1e30, 1e-38), (3e38, 1e-36), (-2e38, 3e-38)])
def test_attention_small_scales_and_large_keys(capi, key, scale):
    """bf16 keys next to the type's end, whose products with a query need more than 32 bits, and scales down to nothing that make logits of them."""
    g = generator(44)
    for q_size in (1.0, 100.0):
        lens, D = [5, 100, 900], 64
        pages, total = table_for(g, lens, 16)
        k, v = pool(g, total, 16, 2, D, torch.bfloat16)
        k.copy_((torch.rand(k.shape, generator=g, device="cuda") * key).to(torch.bfloat16))
        q, out = randn(g, 3, 4, D) * q_size, torch.empty((3, 4, D), device="cuda")
        capi.paged_attention_q8_1(q, k, v, pages, i32(lens), scale=scale, out=out, want_q8=False)
        want, _, far, _ = attended(q, k, v, pages, lens, 16, float(torch.tensor(scale)))
        assert torch.isfinite(out).all() and ((out.double() - want).abs() <= far).all()


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("Hq,Hk,D,page", [(8, 2, 128, 16), (4, 4, 64, 5), (24, 1, 64, 32), (40, 2, 256, 16), (3, 1, 80, 24)])
def test_attention_weights(capi, kind, Hq, Hk, D, page):
    check_attention(capi, generator(Hq + D), kind, Hq, Hk, D, page, [1, 0, 15, 700, 64, 2500], weights=True)


def test_attention_weights_of_another_length(capi):
    """Shorter than the table (tokens behind are attended to, and not counted), longer, and with rows further apart."""
    g = generator(12)
    q, k, v, pages, out = check_attention(capi, g, "f16", 4, 2, 64, 16, [100, 37])
    lens = i32([100, 37])
    whole = torch.zeros((2, 2, pages.shape[1] * 16), device="cuda")
    capi.paged_attention_q8_1(q, k, v, pages, lens, want_q8=False, out=out, weights=whole)
    short, wide = torch.zeros((2, 2, 50), device="cuda"), torch.zeros((2, 2, 400), device="cuda")
    again = torch.empty_like(out)
    capi.paged_attention_q8_1(q, k, v, pages, lens, want_q8=False, out=again, weights=short)
    capi.paged_attention_q8_1(q, k, v, pages, lens, want_q8=False, out=again, weights=wide[..., :77])
    assert torch.equal(again, out)
    assert torch.equal(short, whole[..., :50]) and torch.equal(wide[..., :77], whole[..., :77]) and (wide[..., 77:] == 0).all()
    assert (whole.sum(-1) - 2).abs().max() <= 2 * 200 * U * 2  # two query heads: shares that add up to one each


def test_attention_bad_pages(capi):
    """Tokens on pages that do not exist are not attended to, and reported; a row that has no other pages gives zeros."""
    g = generator(13)
    for page in (16, 4):
        k, v = pool(g, 5, page, 2, 64, torch.float16)
        pages = i32([[0, 5, 1, -3], [-1, -1, -1, -1], [2, 3, 4, 2**31 - 1]])
        lens = [3 * page + 1, 2 * page, 3 * page]
        q, out = randn(g, 3, 4, 64), torch.empty((3, 4, 64), device="cuda")
        xq = capi.paged_attention_q8_1(q, k, v, pages, i32(lens), out=out)
        want, _, far, _ = attended(q, k, v, pages, lens, page, 64**-0.5)
        assert capi.device_fault(clear=True) == capi.FAULT_BAD_PAGE
        assert ((out.double() - want).abs() <= far).all() and (out[1] == 0).all()
        assert torch.equal(xq, capi.quantize_q8_1(out.view(3, 256), capi.ORDER_COL_KSUPER, capi.S_D_SUM_Q))


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("tokens", [3, 40, 3000])
def test_attention_weights_of_bad_pages(capi, kind, tokens):
    """Tokens on pages that do not exist are given nothing: their weights stay as they were, also where a row has no other tokens (in one warp's
    hands, a block's, or several blocks')."""
    g = generator(41)
    need = -(-tokens // 16)
    k, v = pool(g, need + 1, 16, 2, 64, TYPES[kind])
    pages = torch.arange(need, dtype=torch.int32, device="cuda").repeat(3, 1)
    pages[1] = -1
    pages[2, 0] = need + 1
    q, lens = randn(g, 3, 8, 64), i32([tokens] * 3)
    weights = torch.rand((3, 2, need * 16), generator=g, device="cuda")
    before, out = weights.clone(), torch.empty_like(q)
    capi.paged_attention_q8_1(q, k, v, pages, lens, out=out, want_q8=False, weights=weights)
    assert capi.device_fault(clear=True) == capi.FAULT_BAD_PAGE
    assert torch.equal(weights[1], before[1]) and (out[1] == 0).all()
    assert torch.equal(weights[2, :, :16], before[2, :, :16])
    want, shares, far, worst = attended(q, k, v, pages, [tokens] * 3, 16, 64**-0.5)
    assert ((out.double() - want).abs() <= far).all()
    for t in range(3):
        for h in range(2):
            at, share = shares[t][h]
            expect = before[t, h][at].double() + share
            assert ((weights[t, h][at].double() - expect).abs() <= share * worst + expect * 2 * U + 2.0**-120).all()


def test_attention_follows_numbers_that_are_none(capi):
    """NaN among what a row sees makes its heads NaN, and no other row's."""
    g = generator(14)
    k, v = pool(g, 8, 16, 2, 64, torch.float16)
    pages, lens = i32([[0, 1, 2], [3, 4, 5]]), i32([40, 40])
    q, out = randn(g, 2, 4, 64), torch.empty((2, 4, 64), device="cuda")
    k[1, 3, 1] = math.nan
    capi.paged_attention_q8_1(q, k, v, pages, lens, out=out, want_q8=False)
    assert torch.isfinite(out[0, :2]).all() and torch.isnan(out[0, 2:]).all() and torch.isfinite(out[1]).all()


@pytest.mark.parametrize("order", [0, 1])
@pytest.mark.parametrize("s_mode", [0, 1])
def test_attention_blocks_are_the_quantizers(capi, order, s_mode):
    g = generator(15)
    for rows, Hq, Hk, D in ((5, 4, 2, 32), (3, 32, 8, 128), (1, 2, 1, 64), (2, 8, 8, 256), (70, 4, 1, 96)):
        lens = [int(n) for n in torch.randint(0, 300, (rows,), generator=g, device="cuda")]
        pages, total = table_for(g, lens, 16)
        k, v = pool(g, total, 16, Hk, D, torch.bfloat16)
        q, out = randn(g, rows, Hq, D), torch.empty((rows, Hq * D), device="cuda")
        xq = capi.paged_attention_q8_1(q, k, v, pages, i32(lens), out=out, order=order, s_mode=s_mode)
        assert torch.equal(xq, capi.quantize_q8_1(out, order, s_mode))
        assert torch.equal(xq, capi.paged_attention_q8_1(q, k, v, pages, i32(lens), order=order, s_mode=s_mode))  # without fp32


def test_attention_workspace(capi):
    """Calls one after the other in one workspace, of changing lengths, leave its counters zero and give the same bits every time."""
    g = generator(16)
    lens = [3000, 17, 0, 900, 2000]
    pages, total = table_for(g, [3000] * 5, 16)
    k, v = pool(g, total, 16, 2, 128, torch.float16)
    q = randn(g, 5, 8, 128)
    ws = capi.paged_attention_workspace(q, k, pages, weights=True)
    first = {}
    for round_ in range(3):
        for n in ([3000, 17, 0, 900, 2000], [1, 2, 3, 4, 5], [3000] * 5, [0] * 5):
            out, w = torch.empty_like(q), torch.zeros((5, 2, pages.shape[1] * 16), device="cuda")
            capi.paged_attention_q8_1(q, k, v, pages, i32(n), out=out, want_q8=False, weights=w, ws=ws)
            assert (ws[: 4 * 5 * 8] == 0).all()
            if tuple(n) in first:
                assert torch.equal(first[tuple(n)][0], out) and torch.equal(first[tuple(n)][1], w)
            first[tuple(n)] = (out, w)
    with pytest.raises(capi.JqError) as e:
        capi.paged_attention_q8_1(q, k, v, pages, i32(lens), ws=ws[:1024])
    assert e.value.status == capi.ERR_INVALID_ARG
    with pytest.raises(capi.JqError):  # made for calls without weights
        capi.paged_attention_q8_1(q, k, v, pages, i32(lens), weights=w, ws=capi.paged_attention_workspace(q, k, pages))


@pytest.mark.parametrize("made_for", [200, 1])
def test_attention_workspace_of_changing_batches(capi, made_for):
    """A batch that grows and shrinks, and caches of other heads and types, in one workspace: the bits of a workspace of its own each time."""
    g = generator(42)
    calls = []
    for kind, Hq, Hk, D, lens in (("f16", 32, 8, 128, [300] * 200), ("f16", 32, 8, 128, [6000]), ("f16", 32, 8, 128, [3000, 0, 17]),
                                  ("e4m3", 4, 1, 64, [5000, 700]), ("bf16", 16, 2, 128, [40] * 150), ("f16", 32, 8, 128, [1, 900] * 32)):
        pages, total = table_for(g, lens, 16)
        k, v = pool(g, total, 16, Hk, D, TYPES[kind])
        calls.append((randn(g, len(lens), Hq, D), k, v, pages, i32(lens)))
    alone = [torch.full_like(c[0], 9.0) for c in calls]
    for call, out in zip(calls, alone):
        capi.paged_attention_q8_1(*call, out=out, want_q8=False)
    q, k, v, pages, lens = calls[0]
    ws = capi.paged_attention_workspace(q[:made_for], k, pages[:made_for])
    for i in (0, 1, 0, 2, 3, 0, 4, 1, 5, 3, 4, 0):
        out = torch.full_like(alone[i], 9.0)
        capi.paged_attention_q8_1(*calls[i], out=out, want_q8=False, ws=ws)
        assert torch.equal(out, alone[i]), i


def test_attention_in_graphs_and_on_other_streams(capi):
    """Two graphs with workspaces of their own, replayed at once with lengths that change in between; an eager call on a third stream."""
    g = generator(17)
    pages, total = table_for(g, [2000] * 3, 16)
    k, v = pool(g, total, 16, 4, 64, torch.bfloat16)
    q = randn(g, 3, 8, 64)
    lens = [i32([2000, 5, 600]), i32([1, 1999, 0])]
    graphs, outs, streams = [], [torch.empty_like(q) for _ in range(2)], [torch.cuda.Stream() for _ in range(3)]
    spaces = [capi.paged_attention_workspace(q, k, pages) for _ in range(2)]
    torch.cuda.synchronize()
    for i in range(2):
        with torch.cuda.stream(streams[i]):
            capi.paged_attention_q8_1(q, k, v, pages, lens[i], out=outs[i], want_q8=False, ws=spaces[i])
            streams[i].synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=streams[i]):
                capi.paged_attention_q8_1(q, k, v, pages, lens[i], out=outs[i], want_q8=False, ws=spaces[i])
            graphs.append(graph)
    for n in ([[2000, 5, 600], [1, 1999, 0]], [[0, 0, 1], [2000, 2000, 2000]], [[33, 1000, 1], [7, 0, 16]]):
        for i in range(2):
            lens[i].copy_(i32(n[i]))
        torch.cuda.synchronize()
        with torch.cuda.stream(streams[2]):
            eager = torch.empty_like(q)
            capi.paged_attention_q8_1(q, k, v, pages, i32(n[0]), out=eager, want_q8=False)  # makes a workspace of its own
        for _ in range(3):
            for i in range(2):
                with torch.cuda.stream(streams[i]):
                    graphs[i].replay()
        torch.cuda.synchronize()
        for i in range(2):
            alone = torch.empty_like(q)
            capi.paged_attention_q8_1(q, k, v, pages, lens[i], out=alone, want_q8=False)
            assert torch.equal(alone, outs[i])
        assert torch.equal(eager, outs[0])


@pytest.mark.parametrize("want_q8", [False, True])
def test_attention_without_rows(capi, want_q8):
    """As the other calls: a batch that has become empty is no error, whichever outputs are asked for."""
    k, v = pool(generator(20), 2, 16, 2, 64, torch.float16)
    q, out = torch.empty((0, 4, 64), device="cuda"), torch.empty((0, 4, 64), device="cuda")
    for table in (i32([[0, 1]]), torch.empty((0, 2), dtype=torch.int32, device="cuda")):
        capi.paged_attention_q8_1(q, k, v, table, i32([]), out=out, want_q8=want_q8)
        capi.paged_attention_q8_1(q, k, v, table, i32([]), out=out, want_q8=want_q8, weights=torch.empty((0, 2, 32), device="cuda"))


def test_attention_from_strided_queries(capi):
    g = generator(18)
    k, v = pool(g, 4, 16, 2, 64, torch.float16)
    pages, lens = i32([[0, 1], [2, 3]]), i32([20, 32])
    wide = randn(g, 2, 6, 80)
    q = wide[:, 1:5, 8:72]
    one, two = torch.empty((2, 4, 64), device="cuda"), torch.empty((2, 4, 64), device="cuda")
    capi.paged_attention_q8_1(q, k, v, pages, lens, out=one, want_q8=False)
    capi.paged_attention_q8_1(q.contiguous(), k, v, pages, lens, out=two, want_q8=False)
    assert torch.equal(one, two)
    with pytest.raises(capi.JqError) as e:
        capi.paged_attention_q8_1(wide[:, 1:5, 7:71], k, v, pages, lens)
    assert e.value.status == capi.ERR_ALIGN
    with pytest.raises(ValueError):
        capi.paged_attention_q8_1(q, k, v, pages, lens, xq=torch.empty(10, dtype=torch.uint8, device="cuda"))
    with pytest.raises(ValueError):
        capi.paged_attention_q8_1(q, k, v, pages, lens.cpu())


def test_offsets_beyond_32_bits(capi):
    """Pages that begin behind 2^31 elements: written, attended to, and moved."""
    g = generator(19)
    pages_total = (2**31 + 2**22) // (64 * 2 * 128)
    k, v = (torch.zeros((pages_total, 64, 2, 128), dtype=torch.float16, device="cuda") for _ in range(2))
    last = pages_total - 1
    assert last * 64 * 2 * 128 > 2**31
    pages = i32([[last, 3, last - 2]])
    for t in (k, v):
        for p in (last, 3, last - 2):
            t[p] = randn(g, 64, 2, 128).half()
    table, _ = capi.rope_table(128, device="cuda")
    qkv = randn(g, 2, 6 * 128)
    q = capi.rope_append(qkv, i32([9, 10]), table, k, v, pages, i32([150, 5]), seqs=i32([0, 0]))
    assert torch.equal(v[last - 2, 22], qkv.view(2, 6, 128)[0, 4:].half()) and torch.equal(v[last, 5], qkv.view(2, 6, 128)[1, 4:].half())
    out = torch.empty((1, 2, 128), device="cuda")
    capi.paged_attention_q8_1(q[:1], k, v, pages, i32([151]), out=out, want_q8=False)
    want, _, far, _ = attended(q[:1], k, v, pages, [151], 64, 128**-0.5)
    assert ((out.double() - want).abs() <= far).all()
    w = torch.rand((1, 2, 192), generator=g, device="cuda")
    target = i32([[last - 5, last - 6]])
    kept, n = capi.kv_evict(w.clone(), i32([151]), k, v, pages, 100, new_page_table=target)
    for h in range(2):
        for j, i in ((0, kept[0, h, 0].item()), (99, kept[0, h, 99].item())):
            assert torch.equal(k[target[0, j // 64], j % 64, h], k[pages[0, i // 64], i % 64, h])


# ---- eviction --------------------------------------------------------------------------------------------------------------
def chosen(weights, n, keep, recent, sinks):
    """Indices that stay, ascending: plain sorting of Python numbers."""
    if n <= keep:
        return list(range(n))
    stays = set(range(sinks)) | set(range(n - recent, n))
    rest = [i for i in range(n) if i not in stays]
    rest.sort(key=lambda i: (-(-math.inf if math.isnan(weights[i]) else weights[i]), i))
    return sorted(list(stays) + rest[: keep - len(stays)])


def check_evict(capi, g, kind, Hk, D, page, lens, S, keep, recent, sinks, layout="slots", in_place=False, weights=None, same_lens=False, same_weights=None):
    B = len(lens)
    held = [min(max(n, 0), S) for n in lens]
    pages, total = table_for(g, [max(n, min(keep, max(held))) for n in held], page, spare=0)
    new_pages, more = table_for(g, [keep] * B, page, spare=1)
    new_pages = torch.where(new_pages >= 0, new_pages + total, new_pages).to(torch.int32)
    k, v = pool(g, total + more, page, Hk, D, TYPES[kind], layout)
    as_bytes = (lambda t: t.contiguous().view(torch.uint8)) if kind == "e4m3" else (lambda t: t.contiguous().view(torch.int16))
    k0, v0 = as_bytes(k).clone(), as_bytes(v).clone()
    if weights is None:
        weights = torch.rand((B, Hk, S), generator=g, device="cuda")
        weights = torch.where(weights < 0.3, (weights * 20).floor() / 20, weights)  # with ties
    w0 = weights.clone()
    same_weights = in_place if same_weights is None else same_weights
    target = weights if same_weights else torch.full_like(weights, 5.0)
    d_lens = i32(lens)
    kept, new_lens = capi.kv_evict(weights, d_lens, k, v, pages, keep, recent=recent, sinks=sinks, new_page_table=None if in_place else new_pages,
                                   new_weights=target, new_lens=d_lens if same_lens else None)
    if not same_weights:
        assert torch.equal(weights.nan_to_num(), w0.nan_to_num())
    if not same_lens:
        assert d_lens.tolist() == lens
    to = pages if in_place else new_pages
    want_k, want_v = k0.clone(), v0.clone()
    expect = w0.cpu().tolist()
    for b in range(B):
        n = held[b]
        assert new_lens[b].item() == min(n, keep)
        for h in range(Hk):
            stay = chosen(expect[b][h], n, keep, recent, sinks)
            assert kept[b, h].tolist() == stay + [-1] * (keep - len(stay)), (b, h)
            i, j = torch.tensor(stay, device="cuda", dtype=torch.long), torch.arange(len(stay), device="cuda")
            assert torch.equal(target[b, h, : len(stay)].nan_to_num(nan=-9.0), w0[b, h, i].nan_to_num(nan=-9.0)) and (target[b, h, len(stay):] == 0).all()
            old, new = pages[b, i // page].long(), to[b, j // page].long()
            want_k[new, j % page, h] = k0[old, i % page, h]
            want_v[new, j % page, h] = v0[old, i % page, h]
    assert torch.equal(as_bytes(k), want_k) and torch.equal(as_bytes(v), want_v)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("kind,Hk,D,page,layout", [("f16", 2, 64, 16, "slots"), ("bf16", 1, 128, 1, "heads"), ("e4m3", 3, 16, 24, "slots"), ("f16", 2, 80, 5, "both"),
                                                   ("e4m3", 2, 256, 32, "heads"), ("bf16", 4, 256, 7, "both")])
@pytest.mark.parametrize("lens,S,keep,recent,sinks", [
    ([40, 0, 1, 10, 11], 40, 10, 3, 2), ([300, 299, 7], 333, 64, 0, 0), ([100], 100, 1, 0, 0), ([100, 50], 100, 99, 50, 49), ([100, 64, 20], 64, 32, 32, 0),
    ([65, 2000], 2100, 600, 100, 4), ([5000], 5000, 4999, 17, 1), ([9000, 3], 9001, 2049, 1000, 8), ([-5, 30], 30, 8, 8, 0)])
def test_evict(capi, kind, Hk, D, page, layout, lens, S, keep, recent, sinks, in_place):
    check_evict(capi, generator(D + S + keep), kind, Hk, D, page, lens, S, keep, recent, sinks, layout, in_place)


@pytest.mark.parametrize("S", [31, 2048, 2049, 4096, 8200, 16500, 40001])
def test_evict_weights_that_are_hard_to_order(capi, S):
    """All equal, infinities, NaN, both zeros, denormal numbers, negative ones, values that differ in their last bit."""
    g = generator(S)
    odd = torch.tensor([0.0, -0.0, 1.0, 1.0 + 2.0**-23, 1.0 - 2.0**-24, 1e-45, -1e-45, 1e-38, -1.0, math.inf, -math.inf, math.nan, 3e38, -3e38], device="cuda")
    for weights in (torch.zeros((1, 2, S), device="cuda"), odd[torch.randint(0, len(odd), (1, 2, S), generator=g, device="cuda")],
                    torch.full((1, 2, S), math.nan, device="cuda"), (torch.rand((1, 2, S), generator=g, device="cuda") * 2.0**-20 + 1),
                    torch.arange(S, device="cuda").float().expand(1, 2, S).contiguous()):
        for keep, recent, sinks in ((S // 3 + 1, 3, 2), (S - 1, 0, 0)):
            check_evict(capi, g, "f16", 2, 16, 16, [S], S, keep, recent, sinks, weights=weights.clone())


def test_evict_lengths_and_weights_in_place(capi):
    g = generator(23)
    check_evict(capi, g, "f16", 2, 64, 16, [500, 30, 100], 512, 100, 10, 4, same_lens=True)
    check_evict(capi, g, "f16", 2, 64, 16, [500, 30, 100], 512, 100, 10, 4, same_lens=True, in_place=True)
    check_evict(capi, g, "f16", 2, 64, 16, [500, 30, 100], 512, 100, 10, 4, same_weights=True)
    check_evict(capi, g, "f16", 2, 64, 16, [500, 30, 100], 512, 100, 10, 4, in_place=True, same_weights=False)


@pytest.mark.parametrize("in_place", [False, True])
def test_evict_lengths_beyond_the_weights(capi, in_place):
    """They count as the weights' length."""
    check_evict(capi, generator(28), "f16", 2, 64, 16, [400, 33, 2**31 - 1], 300, 100, 9, 3, in_place=in_place)


def test_evict_many_sequences_and_a_long_one(capi):
    check_evict(capi, generator(24), "bf16", 2, 16, 16, [int(n) for n in np.random.default_rng(1).integers(0, 80, 300)], 80, 24, 5, 1)
    check_evict(capi, generator(25), "f16", 1, 16, 64, [300001], 300001, 5000, 100, 4)


def test_evict_bad_pages_and_refusals(capi):
    """A token on a page that does not exist is not moved, and reported; a row of weights longer than a call takes is refused."""
    g = generator(26)
    k, v = pool(g, 6, 4, 1, 16, torch.float16)
    k0, v0 = k.clone(), v.clone()
    w = torch.rand((1, 1, 12), generator=g, device="cuda")
    kept, n = capi.kv_evict(w, i32([12]), k, v, i32([[0, 9, 2]]), 12, new_page_table=i32([[3, 4, -1]]))
    assert capi.device_fault(clear=True) == capi.FAULT_BAD_PAGE
    k0[3], v0[3] = k0[0], v0[0]  # the first page moved; the second has no source, the third no target
    assert torch.equal(k, k0) and torch.equal(v, v0) and n.item() == 12
    most = capi.kv_evict_max_len()
    assert most >= 300001
    too_long = torch.zeros((1, 1, most + 1), device="cuda")
    with pytest.raises(capi.JqError) as e:
        capi.kv_evict(too_long, i32([5]), k, v, i32([[0, 1, 2]]), 4)
    assert e.value.status == capi.ERR_TOO_LARGE
    with pytest.raises(ValueError):
        capi.kv_evict(w, i32([12]), k, v, i32([[0, 1, 2]]), 4, kept=torch.empty((1, 1, 5), dtype=torch.int32, device="cuda"))
    with pytest.raises(ValueError):
        capi.kv_evict(w, i32([12, 3]), k, v, i32([[0, 1, 2]]), 4)


def test_evict_from_pages_that_sequences_share(capi):
    """Two sequences with a common start: each is cut down into pages of its own, and the shared ones stay as they were."""
    g = generator(45)
    k, v = pool(g, 10, 16, 2, 32, torch.float16)
    k0, v0 = k.clone(), v.clone()
    pages, target = i32([[4, 1, 7], [4, 1, 9]]), i32([[0, 2], [3, 5]])
    w = torch.rand((2, 2, 48), generator=g, device="cuda")
    kept, n = capi.kv_evict(w, i32([48, 40]), k, v, pages, 20, recent=4, new_page_table=target, new_weights=torch.empty_like(w))
    assert n.tolist() == [20, 20]
    j = torch.arange(20, device="cuda")
    for b in range(2):
        for h in range(2):
            stay = chosen(w[b, h].tolist(), (48, 40)[b], 20, 4, 0)
            i = torch.tensor(stay, device="cuda")
            assert kept[b, h].tolist() == stay
            for t, t0 in ((k, k0), (v, v0)):
                assert torch.equal(t[target[b, j // 16].long(), j % 16, h], t0[pages[b, i // 16].long(), i % 16, h])
    for t, t0 in ((k, k0), (v, v0)):
        assert torch.equal(t[[1, 4, 6, 7, 8, 9]], t0[[1, 4, 6, 7, 8, 9]])
    with pytest.raises(capi.JqError) as e:
        capi.kv_evict(w, i32([48, 40]), k, v, pages, 20, new_page_table=pages)
    assert e.value.status == capi.ERR_INVALID_ARG


@pytest.mark.parametrize("in_place", [False, True])
def test_evict_budget_next_to_2_31(capi, in_place):
    """The largest budget that is taken: indices one step beyond it have more than 31 bits, and nothing outside the list is written."""
    keep, edge, S = 0x7FFFFF00, 1 << 14, 40
    g = generator(27)
    k, v = pool(g, 7, 16, 1, 16, torch.float16)
    k0, v0 = k.clone(), v.clone()
    pages = i32([[5, 0, 3]])
    new_pages = None
    if not in_place:
        new_pages = torch.full((1, keep // 16), -1, dtype=torch.int32, device="cuda")
        new_pages[0, :3] = i32([6, 2, 1])
    around = torch.full((keep + 2 * edge,), 7, dtype=torch.int32, device="cuda")
    kept = around[edge:edge + keep].view(1, 1, keep)
    w = torch.rand((1, 1, S), generator=g, device="cuda")
    w0 = w.clone()
    _, n = capi.kv_evict(w, i32([S]), k, v, pages, keep, new_page_table=new_pages, kept=kept)
    assert n.item() == S and torch.equal(w, w0)
    assert (around[:edge] == 7).all() and (around[edge + keep:] == 7).all()
    assert kept[0, 0, :S].tolist() == list(range(S)) and kept[0, 0, S:].amax().item() == -1 and kept[0, 0, S:].amin().item() == -1
    if not in_place:
        for old, new, slots in ((5, 6, 16), (0, 2, 16), (3, 1, 8)):
            k0[new, :slots], v0[new, :slots] = k0[old, :slots], v0[old, :slots]
    assert torch.equal(k, k0) and torch.equal(v, v0)


@pytest.mark.parametrize("in_place", [False, True])
def test_append_and_evict_in_graphs_and_on_two_streams(capi, in_place):
    """Recorded and replayed on two streams at once, on caches of their own, with inputs that change in between: the bits of eager calls."""
    g = generator(47)
    B, Hq, Hk, D, page, S, keep = 3, 4, 2, 64, 16, 3000, 700
    table, _ = capi.rope_table(D, device="cuda")
    sides = []
    for i in range(2):
        pages, total = table_for(g, [S] * B, page, spare=0)
        new_pages, more = table_for(g, [keep] * B, page, spare=0)
        k, v = pool(g, total + more, page, Hk, D, torch.float16)
        side = dict(pages=pages, new=None if in_place else new_pages + total, k=k, v=v, w=torch.zeros((B, Hk, S), device="cuda"), lens=i32([0] * B), at=i32([0] * B),
                    qkv=torch.zeros((B, (Hq + 2 * Hk) * D), device="cuda"), q=torch.zeros((B, Hq, D), device="cuda"), kept=i32([[[0] * keep] * Hk] * B),
                    stream=torch.cuda.Stream())
        sides.append(side)

    def step(s):
        capi.rope_append(s["qkv"], s["at"], table, s["k"], s["v"], s["pages"], s["at"], q_out=s["q"])
        capi.kv_evict(s["w"], s["lens"], s["k"], s["v"], s["pages"], keep, recent=50, sinks=4, new_page_table=s["new"], new_lens=s["lens"], kept=s["kept"])

    fields = ("k", "v", "w", "lens", "q", "kept")
    for s in sides:
        with torch.cuda.stream(s["stream"]):
            s["stream"].wait_stream(torch.cuda.default_stream())
            step(s)
            s["stream"].synchronize()
            s["graph"] = torch.cuda.CUDAGraph()
            with torch.cuda.graph(s["graph"], stream=s["stream"]):
                step(s)
    for lens in ([3000, 701, 5], [700, 0, 2999], [1500, 1501, 1]):
        expected = []
        for s in sides:
            s["qkv"].copy_(randn(g, *s["qkv"].shape))
            s["w"].copy_(torch.rand(s["w"].shape, generator=g, device="cuda"))
            s["lens"].copy_(i32(lens))
            s["at"].copy_((i32(lens) - 1).clamp(min=0))
            before = {f: s[f].clone() for f in fields}
            step(s)
            expected.append({f: s[f].clone() for f in fields})
            for f in fields:
                s[f].copy_(before[f])
        torch.cuda.synchronize()
        for s in sides:
            with torch.cuda.stream(s["stream"]):
                s["graph"].replay()
        torch.cuda.synchronize()
        for s, want in zip(sides, expected):
            assert s["lens"].tolist() == [min(n, keep) for n in lens]
            for f in fields:
                assert torch.equal(s[f], want[f]), f


# ---- all of it, the way a decoder uses it --------------------------------------------------------------------------------------
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("graph", [False, True])
def test_decode_steps_of_a_layer(capi, kind, graph):
    """Norm, fused projection, rotation and cache, attention, output projection, step by step for three sequences of their own lengths, with an
    eviction in between; the attention's part is checked against 64 bits on the tensors that went into it."""
    g = generator(31)
    B, Hq, Hk, D, page, hidden = 3, 8, 2, 64, 16, 512
    wide = (Hq + 2 * Hk) * D
    w_qkv = capi.quantize_q4_0(randn(g, wide, hidden) * 0.05)
    w_o = capi.quantize_q4_0(randn(g, hidden, Hq * D) * 0.05)
    norm = torch.rand(hidden, generator=g, device="cuda") + 0.5
    table, mscale = capi.rope_table(D, 10000.0, "wavelength", 4.0, 64, device="cuda")
    S, keep = 96, 40
    pages, total = table_for(g, [S] * B, page)
    k, v = pool(g, total, page, Hk, D, TYPES[kind])
    scale = 0.0625 if kind == "e4m3" else 1.0
    weights = torch.zeros((B, Hk, S), device="cuda")
    # what a loop keeps on the device: positions in the text, and tokens in the cache
    positions, held = i32([30, 7, 0]), i32([30, 7, 0])
    x, xq = randn(g, B, hidden), None
    qkv, q, out, y = (torch.empty((B, n), device="cuda") for n in (wide, Hq * D, Hq * D, hidden))
    lens = torch.empty_like(held)
    hidden_q, out_q = (torch.empty(capi.q8_1_bytes(n, B), dtype=torch.uint8, device="cuda") for n in (hidden, Hq * D))
    ws = capi.paged_attention_workspace(q.view(B, Hq, D), k, pages, weights=True)

    def step():
        capi.rms_norm_q8_1(x, norm, 1e-6, xq=hidden_q)
        capi.mul_mat_q4_0_q8_1(w_qkv, hidden_q, hidden, wide, B, out=qkv)
        capi.rope_append(qkv, positions, table, k, v, pages, held, q_out=q.view(B, Hq, D), mscale=mscale, k_scale=scale, v_scale=scale)
        torch.add(held, 1, out=lens)
        capi.paged_attention_q8_1(q.view(B, Hq, D), k, v, pages, lens, k_scale=scale, v_scale=scale, out=out, weights=weights, xq=out_q, ws=ws)
        capi.mul_mat_q4_0_q8_1(w_o, out_q, Hq * D, hidden, B, out=y)
        held.copy_(lens)
        positions.add_(1)

    replay = step
    if graph:
        state = [t.clone() for t in (positions, held, weights)]
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            step()
            recorded = torch.cuda.CUDAGraph()
            with torch.cuda.graph(recorded, stream=stream):
                step()
        torch.cuda.current_stream().wait_stream(stream)
        for t, s in zip((positions, held, weights), state):
            t.copy_(s)
        replay = recorded.replay
    for i in range(80):  # the longest sequence, 30 tokens to begin with, has no room left after 66 steps
        before = weights.clone()
        x.copy_(randn(g, B, hidden))
        replay()
        n = lens.tolist()
        if i % 7 == 0 or n[0] in (S, keep + 1):
            want, shares, far, worst = attended(q.view(B, Hq, D), k, v, pages, n, page, D**-0.5, k_scale=scale, v_scale=scale)
            assert ((out.view(B, Hq, D).double() - want).abs() <= far).all()
            assert torch.equal(out_q, capi.quantize_q8_1(out, capi.ORDER_COL_KSUPER, capi.S_D_SUM_Q))
            assert torch.equal(y, capi.mul_mat_q4_0_q8_1(w_o, out_q, Hq * D, hidden, B))
            for b in range(B):
                for h in range(Hk):
                    at, share = shares[b][h]
                    expect = before[b, h][at].double() + share
                    assert ((weights[b, h][at].double() - expect).abs() <= share * worst + expect * 2 * U + 2.0**-120).all()
        if n[0] == S:  # the longest has no room left: back to the budget
            kept, _ = capi.kv_evict(weights, held, k, v, pages, keep, recent=16, sinks=4, new_lens=held)
            assert held.tolist() == [min(m, keep) for m in n] and (weights[0, :, keep:] == 0).all()
            assert kept[0, 0, :4].tolist() == [0, 1, 2, 3] and kept[0, 0, -1].item() == S - 1
    assert positions.tolist() == [110, 87, 80] and held.tolist() == [54, 54, 54] and capi.device_fault() == 0
