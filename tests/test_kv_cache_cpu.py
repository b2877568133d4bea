"""What the paged cache's calls compute and refuse without a GPU: where a token lies, tables of rotary positions, arguments."""
import ctypes
import math
import os
import random
import re
import subprocess
import sys
from decimal import Decimal, getcontext

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "jq_kv_cache.h")


class Cache(ctypes.Structure):
    """jq_kv_cache."""

    _fields_ = [("d_k", ctypes.c_void_p), ("d_v", ctypes.c_void_p), ("type", ctypes.c_int)] + \
        [(k, ctypes.c_int64) for k in ("num_pages", "page_size", "num_kv_heads", "head_dim", "stride_page", "stride_slot", "stride_head")] + \
        [("k_scale", ctypes.c_float), ("v_scale", ctypes.c_float), ("d_page_table", ctypes.c_void_p)] + \
        [(k, ctypes.c_int64) for k in ("num_seqs", "max_pages", "table_stride")]


def cache(**changes):
    """A descriptor that is in order (nothing behind its addresses is read on the host), changed."""
    c = dict(d_k=1 << 20, d_v=2 << 20, type=0, num_pages=8, page_size=16, num_kv_heads=2, head_dim=64, stride_page=16 * 128, stride_slot=128,
             stride_head=64, k_scale=1.0, v_scale=1.0, d_page_table=64, num_seqs=3, max_pages=4, table_stride=4)
    return Cache(**{**c, **changes})


def test_every_declared_symbol_is_exported(native_lib):
    text = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    names = sorted(set(re.findall(r"\b(jq_[a-z0-9_]+)\s*\(", text)))
    assert len(names) == 8
    lib = ctypes.CDLL(native_lib.LIB_PATH)
    assert [n for n in names if not hasattr(lib, n)] == []


# ---- where a token lies -------------------------------------------------------------------------------------------
@pytest.fixture(scope="module")
def index(tmp_path_factory):
    """csrc/kv_index.h compiled for the host: (queries on standard input) -> answers."""
    where = tmp_path_factory.mktemp("kv_index")
    (where / "x.cpp").write_text("""
#include <cstdio>
#include "kv_index.h"
int main() {
    long long page_size, token, page, num_pages, sp, ss, max_pages, len;
    while (scanf("%lld %lld %lld %lld %lld %lld %lld %lld", &page_size, &token, &page, &num_pages, &sp, &ss, &max_pages, &len) == 8) {
        jq::KvIndex ix = {};
        ix.stride_page = sp; ix.stride_slot = ss; ix.num_pages = (int32_t)num_pages; ix.max_pages = (int32_t)max_pages;
        jq::kv_set_page_size(ix, (int32_t)page_size);
        printf("%u %lld %d\\n", jq::kv_page_of(ix, (uint32_t)token), (long long)jq::kv_offset(ix, (uint32_t)token, (int32_t)page), jq::kv_length(ix, (int32_t)len));
    }
}
""")
    exe = str(where / "x")
    subprocess.run(["g++", "-O1", "-std=c++17", "-I", os.path.join(ROOT, "jjjetson_ops_b200", "csrc"), str(where / "x.cpp"), "-o", exe], check=True)

    def ask(queries):
        text = "\n".join(" ".join(str(int(v)) for v in q) for q in queries)
        out = subprocess.run([exe], input=text, capture_output=True, text=True, check=True).stdout.split()
        return [tuple(int(v) for v in out[i:i + 3]) for i in range(0, len(out), 3)]

    return ask


def test_page_and_slot_of_a_token(index):
    sizes = list(range(1, 70)) + [127, 128, 129, 1000, 4096, 65537, 10**6 + 3, 2**30 - 1, 2**30, 2**30 + 1, 2**31 - 1]
    queries = []
    for p in sizes:
        for t in {0, 1, p - 1, p, p + 1, 2 * p - 1, 7 * p, 2**31 - 1, (2**31 - 1) // p * p, (2**31 - 1) // p * p - 1}:
            if 0 <= t < 2**31:
                queries.append((p, t, 5, 6, 10**6, 128, 1, 0))
    for (p, t, page, _, sp, ss, _, _), (of, offset, _) in zip(queries, index(queries)):
        assert of == t // p and offset == page * sp + t % p * ss, (p, t)


def test_pages_that_do_not_exist_have_no_place(index):
    for page, there in ((-1, False), (-2**31, False), (0, True), (7, True), (8, False), (2**31 - 1, False)):
        (_, offset, _), = index([(16, 37, page, 8, 2048, 128, 4, 0)])
        assert offset == (page * 2048 + 5 * 128 if there else -1)


def test_offsets_beyond_32_bits(index):
    (_, offset, _), = index([(64, 2**31 - 1, 2**31 - 2, 2**31 - 1, 2**24, 2**17, 1, 0)])
    assert offset == (2**31 - 2) * 2**24 + 63 * 2**17


def test_lengths_are_cut_to_the_table(index):
    for pages, n, want in ((4, 64, 64), (4, 65, 64), (4, 2**31 - 1, 64), (4, -1, 0), (4, -2**31, 0), (0, 5, 0)):
        assert index([(16, 0, 0, 1, 1, 1, pages, n)])[0][2] == want


def test_angles_are_a_quarter_turn_and_a_rest(tmp_path):
    """csrc/kv_index.h compiled for the host: the rest is the exact one to 2^-33 and half a bit, and quarter turns change what sine and cosine are."""
    (tmp_path / "x.cpp").write_text("""
#include <cstdio>
#include "kv_index.h"
int main() {
    unsigned long long steps; int position;
    while (scanf("%llu %d", &steps, &position) == 2) {
        uint32_t quarters;
        const float rest = jq::rope_half_turns(steps, position, &quarters);
        float c = 3, s = 5;
        jq::rope_add_quarters(quarters, &c, &s);
        printf("%u %.17g %g %g\\n", quarters, (double)rest, c, s);
    }
}
""")
    exe = str(tmp_path / "x")
    subprocess.run(["g++", "-O1", "-std=c++17", "-I", os.path.join(ROOT, "jjjetson_ops_b200", "csrc"), str(tmp_path / "x.cpp"), "-o", exe], check=True)
    rng = random.Random(5)
    cases = [(s, p) for s in (0, 1, 2**61 - 1, 2**61, 2**61 + 1, 2**62, 2**63 - 1, 2**63, 2**64 - 2**61, 2**64 - 2**61 - 1, 2**64 - 1)
             for p in (0, 1, -1, 2, 3, -3, 2**31 - 1, -2**31)]
    cases += [(rng.getrandbits(64), rng.randrange(-2**31, 2**31)) for _ in range(2000)]
    out = subprocess.run([exe], input="\n".join("%d %d" % c for c in cases), capture_output=True, text=True, check=True).stdout.split()
    for i, (steps, position) in enumerate(cases):
        quarters, rest, c, s = int(out[4 * i]), float(out[4 * i + 1]), float(out[4 * i + 2]), float(out[4 * i + 3])
        exact = Decimal(steps * position % 2**64) / 2**63 - Decimal(quarters) / 2  # in half turns
        exact = exact - 2 if exact > 1 else exact
        assert abs(exact) <= Decimal("0.25") and abs(rest) <= 0.25 and quarters in (0, 1, 2, 3), (steps, position)
        assert abs(Decimal(rest) - exact) <= Decimal(2) ** -33 + abs(exact) * Decimal(2) ** -24, (steps, position)
        assert (c, s) == ((3, 5), (-5, 3), (-3, -5), (5, -3))[quarters]  # times i for every quarter turn


# ---- rotary tables ------------------------------------------------------------------------------------------------
def _pi():
    getcontext().prec = 60
    x, k = Decimal(0), 0
    for k in range(60):  # Bailey, Borwein and Plouffe's series
        x += (Decimal(4) / (8 * k + 1) - Decimal(2) / (8 * k + 4) - Decimal(1) / (8 * k + 5) - Decimal(1) / (8 * k + 6)) / Decimal(16) ** k
    return x


def test_table_is_the_fraction_of_a_turn(native_lib):
    """Against decimal arithmetic: a step is 2^-64 turns, a frequency in double precision is known to 2^-53 of itself."""
    c, pi = native_lib, _pi()
    given = [1.0, 0.5, 1e-4, 3.0, 7.0, 123456.789, -1.0, -2.5e-3, 0.0, 6.283185307179586, 1e-20]
    table, mscale = c.rope_table(2 * len(given), frequencies=given)
    assert mscale == 1.0 and str(table.dtype) == "torch.int64"
    for f, got in zip(given, table.tolist()):
        turns = Decimal(f) / (2 * pi)
        want = (turns - turns.to_integral_value(rounding="ROUND_FLOOR")) * 2**64
        error = abs(Decimal(got % 2**64) - want)
        error = min(error, 2**64 - error)
        # a long double has 64 bits: the quotient is off by half a step for every turn, taking the whole turns away rounds to half a step
        # (a result next to 1), so does adding the half that rounds, and the rounding itself is off by half a step: 1.5 and |turns| / 2
        assert error <= Decimal("1.5") + abs(turns) * 2, (f, error)


SCALINGS = [("none", 1.0, 0), ("linear", 8.0, 0), ("ntk", 4.0, 0), ("yarn", 16.0, 4096), ("wavelength", 8.0, 8192), ("yarn", 1.0, 64), ("linear", 1.0, 0)]


@pytest.mark.parametrize("rotary", [2, 4, 20, 64, 128, 256])
@pytest.mark.parametrize("how,factor,length", SCALINGS)
def test_scaled_frequencies(native_lib, rotary, how, factor, length):
    base = 10000.0
    table, mscale = native_lib.rope_table(rotary, base, how, factor, length)
    assert len(table) == rotary // 2
    b = base * factor ** (rotary / max(rotary - 2, 1)) if how == "ntk" else base
    for i, got in enumerate(table.tolist()):
        f = b ** (-2.0 * i / rotary)
        if how == "linear":
            f /= factor
        if how == "yarn":
            def pair(turns):
                return rotary * math.log(length / (turns * 2 * math.pi)) / (2 * math.log(base))

            low, high = max(math.floor(pair(32)), 0), min(math.ceil(pair(1)), rotary - 1)
            t = min(max((i - low) / max(high - low, 0.001), 0.0), 1.0)
            f = f / factor * t + f * (1 - t)
        if how == "wavelength":
            t = min(max((length * f / (2 * math.pi) - 1) / 3, 0.0), 1.0)
            f = (1 - t) * f / factor + t * f
        # some ten operations in double precision on each side
        assert abs((got % 2**64) / 2**64 - f / (2 * math.pi)) <= 1e-14 * f + 2**-63, (i, how)
    assert mscale == pytest.approx(0.1 * math.log(factor) + 1 if how == "yarn" else 1.0, rel=2**-23)


@pytest.mark.parametrize("rotary", [2, 20, 128, 1024])
@pytest.mark.parametrize("base", [10000.0, 500000.0, 1.5])
@pytest.mark.parametrize("how,factor", [("none", 1.0), ("linear", 3.0), ("ntk", 4.0), ("wavelength", 8.0), ("yarn", 16.0)])
def test_table_entries_are_rounded_once(native_lib, rotary, base, how, factor):
    """Against decimal arithmetic: a step, 2^-64 turns, is what the entries are off by, not the step of a frequency in double precision, which
    2^31 positions make 2^-25 turns of."""
    pi, length = _pi(), 4096
    r, b, f0 = Decimal(rotary), Decimal(base), Decimal(factor)
    if how == "ntk":
        b *= f0 ** (r / max(r - 2, 1))
    table, _ = native_lib.rope_table(rotary, base, how, factor, length)
    if how == "yarn":
        low, high = ((r * (Decimal(length) / (n * 2 * pi)).ln() / (2 * b.ln())) for n in (32, 1))
        low, high = max(low.to_integral_value(rounding="ROUND_FLOOR"), Decimal(0)), min(high.to_integral_value(rounding="ROUND_CEILING"), r - 1)
    for i, got in enumerate(table.tolist()):
        f = b ** (Decimal(-2 * i) / r)
        t = Decimal(0)
        if how == "linear":
            t = Decimal(1)
        if how == "yarn":
            t = min(max((i - low) / max(high - low, Decimal("0.001")), Decimal(0)), Decimal(1))
        if how == "wavelength":
            t = 1 - min(max((length * f / (2 * pi) - 1) / 3, Decimal(0)), Decimal(1))
        f = f / f0 * t + f * (1 - t)
        # Long doubles have 64 bits, a rounding is 2^-64 of the value: the power's exponent (up to ln(base) of it, with ntk's base some 15), its
        # base, itself, and less than ten operations (where the wavelength's share counts, it is of numbers up to 4): under 50 roundings, 2^-64 each, of
        # at most 2^64 / (2 pi) steps: 8; and 1.5 for the fraction (above)
        error = abs(Decimal(got % 2**64) - f / (2 * pi) * 2**64)
        assert error <= 10, (i, error)


def test_tables_that_are_refused(native_lib):
    c = native_lib
    for args in ((3,), (0,), (-2,), (2048,)):
        with pytest.raises(c.JqError) as e:
            c.rope_table(*args)
        assert e.value.status == c.ERR_SHAPE
    bad = float("nan"), float("inf")
    for kw in ([dict(base=b) for b in (1.0, 0.5, -1.0, *bad)] + [dict(scaling="linear", factor=f) for f in (0.5, 0.0, -1.0, *bad)] +
               [dict(scaling=s, factor=2.0) for s in ("yarn", "wavelength")] + [dict(scaling="ntk", factor=1e300)] +
               [dict(frequencies=[1.0] * 31 + [b]) for b in bad]):
        with pytest.raises(c.JqError) as e:
            c.rope_table(64, **kw)
        assert e.value.status == c.ERR_INVALID_ARG, kw
    for kw in (dict(scaling="other"), dict(frequencies=[1.0])):
        with pytest.raises(ValueError):
            c.rope_table(64, **kw)


# ---- refusals of the C calls: none of these reaches the device ---------------------------------------------------------
BAD_CACHES = [
    ("ERR_INVALID_ARG", dict(type=3)), ("ERR_INVALID_ARG", dict(type=-1)), ("ERR_INVALID_ARG", dict(num_pages=0)), ("ERR_INVALID_ARG", dict(page_size=0)),
    ("ERR_INVALID_ARG", dict(num_kv_heads=0)), ("ERR_INVALID_ARG", dict(num_seqs=-1)), ("ERR_INVALID_ARG", dict(max_pages=-1)),
    ("ERR_SHAPE", dict(head_dim=0)), ("ERR_SHAPE", dict(head_dim=24)), ("ERR_SHAPE", dict(head_dim=272)),
    ("ERR_TOO_LARGE", dict(num_pages=2**31)), ("ERR_TOO_LARGE", dict(max_pages=2**28, table_stride=2**28)), ("ERR_TOO_LARGE", dict(num_kv_heads=2**16)),
    ("ERR_INVALID_ARG", dict(d_k=None)), ("ERR_INVALID_ARG", dict(d_v=None)), ("ERR_INVALID_ARG", dict(d_page_table=None)),
    ("ERR_INVALID_ARG", dict(table_stride=3)), ("ERR_INVALID_ARG", dict(stride_slot=32)), ("ERR_INVALID_ARG", dict(stride_head=0)),
    ("ERR_INVALID_ARG", dict(stride_page=-2048)), ("ERR_ALIGN", dict(stride_slot=132)), ("ERR_ALIGN", dict(d_k=(1 << 20) + 8)),
    ("ERR_ALIGN", dict(d_v=(2 << 20) + 2)), ("ERR_ALIGN", dict(d_page_table=66)), ("ERR_TOO_LARGE", dict(stride_page=2**60)),
    ("ERR_INVALID_ARG", dict(k_scale=0.0)), ("ERR_INVALID_ARG", dict(v_scale=-1.0)), ("ERR_INVALID_ARG", dict(k_scale=float("nan"))),
    ("ERR_INVALID_ARG", dict(v_scale=float("inf"))),
]


def _append(c, lib, rows=2, q_heads=4, rotary=64, mscale=1.0, qkv=64, q=64, positions=64, idx=64, seqs=None, table=64, stride=8 * 64, q_stride=256,
            q_head=64, descriptor=None):
    d = cache() if descriptor is None else descriptor
    return lib.jq_rope_kv_append_device(None, qkv, stride, q, q_stride, q_head, positions, idx, seqs, table, rotary, rows, q_heads, ctypes.byref(d), 0, mscale)


def _attend(c, lib, rows=2, q_heads=4, q=64, lens=64, seqs=None, scale=0.1, window=0, out=64, xq=None, order=1, s_mode=1, weights=None, stride=0,
            length=0, ws=64, ws_bytes=1 << 40, q_stride=256, q_head=64, descriptor=None):
    d = cache() if descriptor is None else descriptor
    return lib.jq_paged_attention_q8_1_device(None, q, q_stride, q_head, rows, q_heads, ctypes.byref(d), lens, seqs, scale, window, out, xq, order, s_mode,
                                              weights, stride, length, ws, ws_bytes)


def _evict(c, lib, lens=64, weights=64, stride=64, max_len=64, keep=8, recent=2, sinks=1, new_table=None, new_pages=0, new_stride=0, kept=64, new_lens=64,
           new_weights=128, new_weights_stride=64, descriptor=None):
    d = cache() if descriptor is None else descriptor
    return lib.jq_kv_evict_device(None, ctypes.byref(d), lens, weights, stride, max_len, keep, recent, sinks, new_table, new_pages, new_stride, kept, new_lens,
                                  new_weights, new_weights_stride)


@pytest.mark.parametrize("status,change", BAD_CACHES)
def test_bad_caches_are_refused_by_every_call(native_lib, status, change):
    c, lib = native_lib, native_lib.lib()
    bad = cache(**change)
    want = getattr(c, status)
    for call in (_append, _attend, _evict):
        assert call(c, lib, descriptor=bad) == want, (call.__name__, c.last_error())
    assert lib.jq_paged_attention_ws_bytes(2, 4, ctypes.byref(bad), 0) == 0
    assert lib.jq_rope_kv_append_device(None, 64, 512, 64, 256, 64, 64, 64, None, 64, 64, 2, 4, None, 0, 1.0) == c.ERR_INVALID_ARG


@pytest.mark.parametrize("status,call,args", [
    ("ERR_SHAPE", _append, dict(rotary=0)), ("ERR_SHAPE", _append, dict(rotary=3)), ("ERR_SHAPE", _append, dict(rotary=66)),
    ("ERR_INVALID_ARG", _append, dict(rows=-1)), ("ERR_INVALID_ARG", _append, dict(mscale=float("nan"))), ("ERR_INVALID_ARG", _append, dict(qkv=None)),
    ("ERR_INVALID_ARG", _append, dict(q=None)), ("ERR_INVALID_ARG", _append, dict(positions=None)), ("ERR_INVALID_ARG", _append, dict(idx=None)),
    ("ERR_INVALID_ARG", _append, dict(table=None)), ("ERR_ALIGN", _append, dict(qkv=66)), ("ERR_ALIGN", _append, dict(table=68)),
    ("ERR_ALIGN", _append, dict(seqs=65)), ("ERR_INVALID_ARG", _append, dict(stride=511)), ("ERR_INVALID_ARG", _append, dict(q_stride=63)),
    ("ERR_INVALID_ARG", _append, dict(q_head=32)), ("OK", _append, dict(rows=0)),
    ("ERR_SHAPE", _attend, dict(q_heads=3)), ("ERR_INVALID_ARG", _attend, dict(q_heads=0)), ("ERR_INVALID_ARG", _attend, dict(window=-1)),
    ("ERR_INVALID_ARG", _attend, dict(scale=float("inf"))), ("ERR_INVALID_ARG", _attend, dict(out=None)), ("ERR_INVALID_ARG", _attend, dict(rows=4)),
    ("ERR_INVALID_ARG", _attend, dict(xq=64, order=2)), ("ERR_INVALID_ARG", _attend, dict(xq=64, s_mode=5)),
    ("ERR_UNSUPPORTED", _attend, dict(xq=64, descriptor=cache(head_dim=48, stride_head=48, stride_slot=96))),
    ("ERR_UNSUPPORTED", _attend, dict(xq=64, q_heads=3, descriptor=cache(num_kv_heads=1))),
    ("ERR_TOO_LARGE", _attend, dict(rows=3, descriptor=cache(page_size=2**10, max_pages=2**21 - 1, table_stride=2**21, num_kv_heads=4, stride_page=2**18))),
    ("ERR_TOO_LARGE", _attend, dict(rows=2**27 - 1, seqs=64, weights=None, descriptor=cache(max_pages=2**26, table_stride=2**26))),
    ("ERR_UNSUPPORTED", _attend, dict(weights=64, seqs=64)), ("ERR_INVALID_ARG", _attend, dict(weights=64, stride=3, length=4)),
    ("ERR_INVALID_ARG", _attend, dict(weights=64, length=-1)),
    ("ERR_INVALID_ARG", _attend, dict(q=None)), ("ERR_INVALID_ARG", _attend, dict(lens=None)), ("ERR_INVALID_ARG", _attend, dict(ws=None)),
    ("ERR_ALIGN", _attend, dict(q=72)), ("ERR_ALIGN", _attend, dict(out=72)), ("ERR_ALIGN", _attend, dict(xq=72)), ("ERR_ALIGN", _attend, dict(ws=72)),
    ("ERR_ALIGN", _attend, dict(q_stride=257)), ("ERR_ALIGN", _attend, dict(q_head=66)), ("ERR_ALIGN", _attend, dict(lens=66)), ("OK", _attend, dict(rows=0)),
    ("ERR_INVALID_ARG", _evict, dict(keep=0)), ("ERR_INVALID_ARG", _evict, dict(recent=-1)), ("ERR_INVALID_ARG", _evict, dict(sinks=-1)),
    ("ERR_INVALID_ARG", _evict, dict(recent=8)), ("ERR_INVALID_ARG", _evict, dict(sinks=9, recent=0)), ("ERR_INVALID_ARG", _evict, dict(max_len=-1)),
    ("ERR_TOO_LARGE", _evict, dict(max_len=1 << 30, stride=1 << 30, new_weights_stride=1 << 30)), ("ERR_INVALID_ARG", _evict, dict(stride=63)),
    ("ERR_INVALID_ARG", _evict, dict(new_weights_stride=63)), ("ERR_INVALID_ARG", _evict, dict(lens=None)), ("ERR_INVALID_ARG", _evict, dict(kept=None)),
    ("ERR_INVALID_ARG", _evict, dict(weights=None)), ("ERR_INVALID_ARG", _evict, dict(new_weights=None)), ("ERR_INVALID_ARG", _evict, dict(new_lens=None)),
    ("ERR_ALIGN", _evict, dict(weights=66)), ("ERR_INVALID_ARG", _evict, dict(new_weights=64, new_weights_stride=65)),
    ("ERR_INVALID_ARG", _evict, dict(new_table=64, new_pages=0)), ("ERR_INVALID_ARG", _evict, dict(new_table=64, keep=33, new_pages=2, new_stride=2)),
    ("ERR_INVALID_ARG", _evict, dict(new_table=64, new_pages=2, new_stride=1)), ("OK", _evict, dict(descriptor=cache(num_seqs=0))),
])
def test_refused_arguments(native_lib, status, call, args):
    c = native_lib
    assert call(c, c.lib(), **args) == getattr(c, status), c.last_error()


def test_eviction_refuses_the_own_table_as_the_new_one(native_lib):
    """Tokens would move to pages that others are still read from."""
    c, lib = native_lib, native_lib.lib()
    own = cache()
    assert _evict(c, lib, new_table=own.d_page_table, new_pages=4, new_stride=4, descriptor=own) == c.ERR_INVALID_ARG
    assert "own" in c.last_error()


def test_calls_without_rows_need_no_buffers(native_lib):
    """Empty tensors have no address: which of them there are does not matter."""
    c, lib = native_lib, native_lib.lib()
    assert _attend(c, lib, rows=0, out=None) == c.OK
    assert _attend(c, lib, rows=0, out=None, q=None, lens=None, ws=None) == c.OK
    assert _attend(c, lib, rows=0, out=None, xq=64) == c.OK
    assert _append(c, lib, rows=0, qkv=None, q=None, positions=None, idx=None) == c.OK
    assert _attend(c, lib, rows=0, window=-1) == c.ERR_INVALID_ARG


def test_workspaces_that_would_overflow_are_refused(native_lib):
    """Sizes whose product has more than 64 bits: an error, not a small number."""
    lib = native_lib.lib()
    wide = cache(num_kv_heads=65535, page_size=2**10, max_pages=2**21 - 1, table_stride=2**21, stride_page=2**40)
    for rows in (1, 65535, 2**27 - 1):
        assert lib.jq_paged_attention_ws_bytes(rows, 65535, ctypes.byref(wide), 1) == 0
        assert native_lib.last_error()


def test_plain_rope_refuses(native_lib):
    c, lib = native_lib, native_lib.lib()

    def call(x=64, out=64, positions=64, table=64, rows=2, heads=3, dim=64, rotary=32, xr=192, xh=64, outr=192, outh=64, mscale=1.0):
        return lib.jq_rope_device(None, x, out, positions, table, rows, heads, dim, rotary, xr, xh, outr, outh, 0, mscale)

    assert call(rows=0) == c.OK and call(heads=0) == c.OK
    for kw in (dict(dim=63, rotary=32), dict(dim=1026), dict(rotary=0), dict(rotary=33), dict(rotary=66)):
        assert call(**kw) == c.ERR_SHAPE, kw
    for kw in (dict(rows=-1), dict(heads=-1), dict(x=None), dict(out=None), dict(positions=None), dict(table=None), dict(outr=63), dict(outh=63),
               dict(mscale=float("inf"))):
        assert call(**kw) == c.ERR_INVALID_ARG, kw
    for kw in (dict(x=65), dict(out=66), dict(positions=67), dict(table=68)):
        assert call(**kw) == c.ERR_ALIGN, kw


# ---- refusals of the tensor calls, on tensors without memory --------------------------------------------------------
TENSORS = """
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from jjjetson_ops_b200 import capi as c

def t(*shape, dtype=torch.float32):
    return torch.empty(shape, device="cuda", dtype=dtype)
i32, f16, f64 = torch.int32, torch.float16, torch.float64
def kv(pages=4, slots=16, heads=2, dim=64, dtype=f16):
    return t(pages, slots, heads, dim, dtype=dtype)
def attend(q=None, k=None, v=None, table=None, lens=None, **kw):
    return c.paged_attention_q8_1(t(3, 4, 64) if q is None else q, kv() if k is None else k, kv() if v is None else v,
                                  t(3, 2, dtype=i32) if table is None else table, t(3, dtype=i32) if lens is None else lens,
                                  **{**dict(ws=t(4096, dtype=torch.uint8), out=t(3, 4, 64), want_q8=False), **kw})
"""


def _raised(calls):
    code = TENSORS + "for call in %r:\n    with FakeTensorMode():\n        try:\n            eval(call)\n            print('nothing')\n" \
        "        except Exception as e:\n            print(type(e).__name__)\n" % (calls,)
    r = subprocess.run([sys.executable, "-W", "ignore", "-c", code], capture_output=True, text=True, cwd=ROOT, timeout=300)
    assert r.returncode == 0, (r.returncode, r.stdout, r.stderr[-2000:])
    return r.stdout.split()


def test_tensors_that_are_refused(native_lib):
    calls = [
        "c.rope(t(3, 64), t(3, dtype=i32), t(32, dtype=torch.int64), out=t(3, 64))",
        "c.rope(t(3, 2, 64, dtype=f16), t(3, dtype=i32), t(32, dtype=torch.int64))",
        "c.rope(t(3, 64, 2).transpose(1, 2), t(3, dtype=i32), t(32, dtype=torch.int64), out=t(3, 2, 64))",
        "c.rope(t(3, 2, 64), t(3, dtype=torch.int64), t(32, dtype=torch.int64))",
        "c.rope(t(3, 2, 64), t(4, dtype=i32), t(32, dtype=torch.int64))",
        "c.rope(t(3, 2, 64), t(3, dtype=i32), t(32))",
        "c.rope_append(t(3, 512), t(3, dtype=i32), t(32, dtype=torch.int64), kv(dtype=f64), kv(), t(3, 2, dtype=i32), t(3, dtype=i32))",
        "c.rope_append(t(3, 512), t(3, dtype=i32), t(32, dtype=torch.int64), kv(), kv(dtype=torch.bfloat16), t(3, 2, dtype=i32), t(3, dtype=i32))",
        "c.rope_append(t(3, 512), t(3, dtype=i32), t(32, dtype=torch.int64), kv(), kv(pages=5), t(3, 2, dtype=i32), t(3, dtype=i32))",
        "c.rope_append(t(3, 512), t(3, dtype=i32), t(32, dtype=torch.int64), kv(), kv().transpose(1, 2).contiguous().transpose(1, 2), t(3, 2, dtype=i32), t(3, dtype=i32))",
        "c.rope_append(t(3, 512), t(3, dtype=i32), t(32, dtype=torch.int64), kv().transpose(2, 3), kv(), t(3, 2, dtype=i32), t(3, dtype=i32))",
        "c.rope_append(t(3, 512), t(3, dtype=i32), t(32, dtype=torch.int64), kv(), kv(), t(3, 2), t(3, dtype=i32))",
        "attend(q=t(3, 4, 32))",
        "attend(q=t(3, 256))",
        "attend(k=None, v=kv(heads=3))",
        "attend(table=t(6, dtype=i32))",
        "attend(lens=t(3, 1, dtype=i32))",
        "attend(k=[0])",
        "c.kv_evict(t(3, 2, 30, dtype=f16), t(3, dtype=i32), kv(), kv(), t(3, 2, dtype=i32), 8, kept=t(3, 2, 8, dtype=i32))",
        "c.kv_evict(t(3, 30), t(3, dtype=i32), kv(), kv(), t(3, 2, dtype=i32), 8, kept=t(3, 2, 8, dtype=i32))",
    ]
    assert _raised(calls) == ["ValueError"] * len(calls)


def test_tensors_without_memory_are_a_runtime_error(native_lib):
    """An exception, not the end of the process."""
    calls = [
        "torch.vmap(lambda v: c.rope(v, t(3, dtype=i32), t(32, dtype=torch.int64), out=t(3, 2, 64)))(t(5, 3, 2, 64))",
        "torch.vmap(lambda v: attend(q=v))(t(5, 3, 4, 64))",
        "torch.vmap(lambda v: c.kv_evict(v, t(3, dtype=i32), kv(), kv(), t(3, 2, dtype=i32), 8, kept=t(3, 2, 8, dtype=i32), new_lens=t(3, dtype=i32)))(t(5, 3, 2, 30))",
    ]
    got = _raised(calls)
    assert all(g in ("RuntimeError", "DataDependentOutputException", "NotImplementedError") for g in got), got
