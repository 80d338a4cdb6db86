"""The paged int8 cache without a GPU: its index arithmetic compiled for the host, the refusals of its three ops, and the
argument handling of PagedKvInt8."""
import ctypes as C
import os
import re
import subprocess

import numpy as np
import pytest
import torch

from kaio_b200 import _lib
from kaio_b200.kv_cache import PagedKvInt8

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def run_cpp(tmp_path, text):
    src, exe = tmp_path / "t.cpp", tmp_path / "t"
    src.write_text(text)
    subprocess.run(["g++", "-O1", "-std=c++17", "-fsanitize=undefined", "-fno-sanitize-recover", "-I",
                    os.path.join(ROOT, "kaio_b200", "csrc"), str(src), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout + r.stderr


def test_every_row_is_in_one_span_whatever_the_split(tmp_path):
    """The units of a grid, searched and cut as the kernels do it, hold every new token once and its position with it; batches of
    1 to 1100 sequences, lengths of zero among them."""
    run_cpp(tmp_path, r'''
#include <initializer_list>
#include <random>
#include <vector>
#include "kv_index.cuh"
using namespace kaio;
int main()
{
    std::mt19937 rng(7);
    for (uint32_t batch : {1u, 2u, 31u, 32u, 33u, 100u, 1100u})
        for (int mode = 0; mode < 4; ++mode) {
            std::vector<int32_t> start(batch + 1, 0), kv(batch);
            for (uint32_t b = 0; b < batch; ++b) {
                const int n = mode == 0 ? 1 : mode == 1 ? rng() % 2 : mode == 2 ? rng() % 70 : (rng() % 5 ? 0 : rng() % 300);
                start[b + 1] = start[b] + n;
                kv[b] = n + rng() % 100;
            }
            const uint32_t rows = start[batch] + rng() % 20;  // some belong to no sequence
            std::vector<int> seen(rows + 1, 0);
            for (uint32_t u = 0; u < rows / 16 + 2 * batch; ++u) {
                KvSearch s = {0, batch};
                while (s.n > 1) {
                    uint32_t hits = 0;
                    for (uint32_t lane = 0; lane < 32; ++lane) {
                        const uint32_t at = lane * s.step();
                        if (at < s.n && kv_first_unit(start[s.lo + at], s.lo + at, 1, 4, 2) <= u)
                            hits |= 1u << lane;
                    }
                    s.narrow(hits);
                }
                const uint32_t b = s.lo, local = u - kv_first_unit(start[b], b, 1, 4, 2);
                const KvSpan p = kv_append_span(start[b], start[b + 1], kv[b], rows, local);
                if (p.bad)
                    return 1;
                for (uint32_t slot = p.begin; slot < p.end; ++slot) {
                    const uint32_t row = p.row0 + slot;
                    if (row < (uint32_t)start[b] || row >= (uint32_t)start[b + 1] || seen[row]++)
                        return 2;
                    if (p.base + slot != (uint32_t)kv[b] - (start[b + 1] - row))
                        return 3;
                }
            }
            for (int r = 0; r < start[batch]; ++r)
                if (seen[r] != 1)
                    return 4;
        }
    return 0;
}
''')


def test_bad_numbers_lead_nowhere(tmp_path):
    """Row starts, lengths and pages of every sign and size: no row, table entry or page outside its buffer comes out."""
    run_cpp(tmp_path, r'''
#include <cstdint>
#include <initializer_list>
#include "kv_index.cuh"
using namespace kaio;
int main()
{
    const int32_t v[] = {INT32_MIN, -17, -1, 0, 1, 5, 16, 31, 100, 1000, INT32_MAX - 1, INT32_MAX};
    const uint32_t rows = 100;
    for (int32_t q0 : v) for (int32_t q1 : v) for (int32_t kv : v)
        for (uint32_t local : {0u, 1u, 6u, 0x0fffffffu, 0xfffffff0u, 0xffffffffu}) {
            const KvSpan s = kv_append_span(q0, q1, kv, rows, local);
            if (s.bad && s.end)
                return 1;
            if ((q0 < 0 || q1 < q0 || q1 > 100) && s.bad != KV_SITE_ROWS)
                return 2;
            if (s.end > KV_BLOCK)
                return 3;
            for (uint32_t slot = s.begin; slot < s.end; ++slot)
                if (s.row0 + slot >= rows || s.row0 + slot < (uint32_t)q0 || s.row0 + slot >= (uint32_t)q1)
                    return 4;
        }
    for (uint32_t shift : {4u, 8u}) for (uint32_t pos : {0u, 15u, 16u, 159u, 160u, 0x7fffffffu, 0xffffffffu})
        for (uint32_t b : {0u, 2u, 3u, 0xffffffffu}) {
            const uint64_t at = kv_table_entry(b, pos, shift, 10, 3);
            if (at > 30 || (at < 30) != (b < 3 && pos >> shift < 10))
                return 5;
        }
    for (int32_t e : v) {
        const uint32_t p = kv_checked_page(e, 32);
        if (p != KV_NO_PAGE && p >= 32)
            return 6;
        if ((e >= 0 && e < 32) != (p != KV_NO_PAGE))
            return 7;
    }
    return 0;
}
''')


def test_the_cut_of_units_over_workers(tmp_path):
    """Every unit has one worker, ranges and owners agree; a sequence's numbers are taken or refused as a whole."""
    run_cpp(tmp_path, r'''
#include <initializer_list>
#include "kv_index.cuh"
using namespace kaio;
int main()
{
    for (uint32_t workers : {1u, 3u, 148u, 1184u, 1280u})
        for (uint64_t units : {1ull, 2ull, 147ull, 148ull, 149ull, 1183ull, 1184ull, 5000ull, 99991ull, 1ull << 33}) {
            const KvCut c(units, workers);
            if (c.workers > workers || c.workers > units || c.begin(0) != 0 || c.begin(c.workers) != units)
                return 1;
            for (uint32_t w = 0; w < c.workers; ++w) {
                const uint64_t lo = c.begin(w), hi = c.begin(w + 1);
                if (lo >= hi)
                    return 2;
                for (uint64_t u : {lo, (lo + hi) / 2, hi - 1})
                    if (c.owner(u) != w)
                        return 3;
            }
        }
    const int32_t v[] = {INT32_MIN, -1, 0, 1, 3, 100, INT32_MAX};
    for (int32_t q0 : v) for (int32_t q1 : v) for (int32_t kv : v) {
        const KvSequence s = kv_sequence(q0, q1, kv, 100, 3, 64);
        const bool rows = q0 >= 0 && q1 >= q0 && q1 <= 100;
        if (s.new_tokens && (!rows || q0 + s.new_tokens > 100 || s.new_tokens > 3 || s.kv > 64 || s.bad))
            return 4;
        if (rows && q1 == q0 && (s.bad || s.new_tokens))
            return 5;
        if (!rows && s.bad != KV_SITE_ROWS)
            return 6;
        for (uint32_t i = 0; i < s.new_tokens; ++i) {
            const int64_t want = (int64_t)s.kv - s.new_tokens + i + 1;
            if (kv_visible(s, i, true) != (want > 0 ? want : 0) || kv_visible(s, i, false) != s.kv)
                return 7;
        }
    }
    return 0;
}
''')


@pytest.fixture(scope="module")
def lib():
    from kaio_b200 import build
    build.build()
    return _lib.load()


# one page of 16 tokens, one head of 64, one sequence, one token
SIZES = dict(batch=1, tokens=1, max_new=1, heads=2, kv_heads=1, head_dim=64, q_stride=128, kv_stride=64, rot_dim=64, interleaved=0,
             max_pos=16, page_size=16, num_pages=1, max_pages=1, causal=1)
LENS = dict(q=128, k=64, v=64, cos=512, sin=512, q_out=128, k_cache=1024, v_cache=1024, k_scale=1, v_scale=1, block_table=1,
            q_start=2, kv_start=2, kv_len=1, k_out=64, v_out=64, out=128, scratch=1 << 24)
P = 0x10000  # an address that is never followed: every call below is refused first
ORDER = {
    "rope_append_kv_int8": ("q k v cos sin q_out k_cache v_cache k_scale v_scale block_table q_start kv_len",
                            "batch tokens heads kv_heads head_dim q_stride kv_stride rot_dim interleaved max_pos page_size num_pages max_pages"),
    "gather_kv_int8": ("k_cache v_cache k_scale v_scale block_table kv_start k_out v_out",
                       "batch tokens kv_heads head_dim page_size num_pages max_pages"),
    "attention_paged_int8": ("q k_cache v_cache k_scale v_scale block_table q_start kv_len out scratch",
                             "batch tokens max_new heads kv_heads head_dim q_stride causal page_size num_pages max_pages"),
}
ALL = tuple(ORDER)


def refused(lib, op, text, null=(), odd=(), **other):
    bufs, sizes = ORDER[op]
    args = []
    for name in bufs.split():
        args += [None if name in null else P + (2 if name in odd else 0), other.get(name + "_len", LENS[name])]
    args += [other.get(name, SIZES[name]) for name in sizes.split()]
    rc = getattr(lib, "kaio_b200_" + op)(*args, None)
    message = lib.kaio_b200_last_error().decode()
    assert rc == 1 and message.startswith(op) and text in message, (rc, message)


@pytest.mark.parametrize("op", ALL)
def test_refusals_of_the_cache(lib, op):
    for name in ("batch", "tokens", "kv_heads", "num_pages", "max_pages"):
        refused(lib, op, "dimensions must be non-zero", **{name: 0})
    refused(lib, op, "batch must be ≤ 32768 (got 32769)", batch=32769)
    for d in (0, 32, 65, 96, 256):
        refused(lib, op, "head_dim must be 64 or 128", head_dim=d)
    for page in (0, 8, 24, 512):
        refused(lib, op, "page_size must be 16, 32, 64, 128 or 256", page_size=page)
    refused(lib, op, "num_pages*kv_heads*page_size must fit 31 bits", num_pages=1 << 27)
    refused(lib, op, "max_pages*page_size must fit 31 bits", max_pages=1 << 27)
    refused(lib, op, "batch*max_pages*page_size must be ≤ 2^37", max_pages=1 << 20, batch=1 << 14)
    for name, kind in (("k_cache", "K cache too small: need 1024 i8"), ("v_cache", "V cache too small"), ("k_scale", "K scales too small"),
                       ("v_scale", "V scales too small"), ("block_table", "block_table too small: need 1 i32 (1×1), got 0")):
        refused(lib, op, kind, **{name + "_len": LENS[name] - 1})
    start = "kv_start" if op == "gather_kv_int8" else "q_start"
    refused(lib, op, f"{start} too small: need 2 i32, got 1", **{start + "_len": 1})
    for name, kind in (("k_cache", "K cache"), ("v_cache", "V cache"), ("k_scale", "K scales"), ("block_table", "block_table"), (start, start)):
        refused(lib, op, f"{kind} pointer is null", null=(name,))
    refused(lib, op, "caches must be 16-byte aligned", odd=("v_cache",))
    if op != "gather_kv_int8":
        refused(lib, op, "heads (3) must be a multiple of kv_heads (2)", heads=3, kv_heads=2)
        refused(lib, op, "kv_len too small: need 1 i32, got 0", kv_len_len=0)
        refused(lib, op, "kv_len pointer is null", null=("kv_len",))
        refused(lib, op, "at most 32768 query heads", heads=32769)


def test_refusals_of_the_append(lib):
    op = "rope_append_kv_int8"
    refused(lib, op, "the row stride of K (63) must be at least 64", kv_stride=63)
    refused(lib, op, "the row stride of Q (127) must be at least 128", q_stride=127)
    refused(lib, op, "multiple of 8 (got 68)", kv_stride=68)
    for name, text in (("k", "K buffer too small: need 64 f16, got 63"), ("v", "V buffer too small"), ("q", "Q buffer too small: need 128 f16"),
                       ("q_out", "q_out buffer too small"), ("cos", "cos too small: need 512 f32 (16×32), got 511"), ("sin", "sin too small")):
        refused(lib, op, text, **{name + "_len": LENS[name] - 1})
    refused(lib, op, "K buffer too small: need 192 f16", tokens=3, kv_stride=64)
    refused(lib, op, "Q and q_out go together", null=("q",))
    refused(lib, op, "Q and q_out go together", null=("q_out",))
    refused(lib, op, "q_out may be Q itself only when", q_stride=136, q_len=1000)
    refused(lib, op, "dimensions must be non-zero", heads=0)
    for rot in (8, 24, 80):
        refused(lib, op, "rot_dim must be a multiple of 16 up to head_dim", rot_dim=rot)
    refused(lib, op, "max_pos must be non-zero", max_pos=0)
    refused(lib, op, "cos pointer is null", null=("cos",))
    for name, text in (("q", "Q must be 16-byte aligned"), ("k", "K must be"), ("v", "V must be"), ("q_out", "q_out must be"),
                       ("sin", "cos and sin must be 16-byte aligned")):
        refused(lib, op, text, odd=(name,))


def test_refusals_of_the_others(lib):
    for name in ("k_out", "v_out"):
        refused(lib, "gather_kv_int8", f"{name} buffer too small: need 64 f16, got 63", **{name + "_len": 63})
        refused(lib, "gather_kv_int8", f"{name} pointer is null", null=(name,))
        refused(lib, "gather_kv_int8", f"{name} must be 16-byte aligned", odd=(name,))
    op = "attention_paged_int8"
    refused(lib, op, "dimensions must be non-zero", max_new=0)
    refused(lib, op, "the row stride of Q (120) must be at least 128", q_stride=120)
    refused(lib, op, "Q buffer too small", q_len=127)
    refused(lib, op, "out buffer too small", out_len=127)
    for name in ("q", "out"):
        refused(lib, op, "pointer is null", null=(name,))
        refused(lib, op, "must be 16-byte aligned", odd=(name,))
    n = C.c_size_t(7)
    assert lib.kaio_b200_attention_paged_int8_scratch(1, 1, 1, 32, 32, 96, C.byref(n)) == 1
    assert lib.kaio_b200_attention_paged_int8_scratch(1, 1, 1, 32, 0, 128, C.byref(n)) == 1
    assert lib.kaio_b200_attention_paged_int8_scratch(1, 1, 1, 32, 32, 128, None) == 1
    assert n.value == 7
    for sizes in ((1, 1, 1, 32, 32, 128), (64, 64, 1, 64, 8, 128), (1, 512, 512, 64, 8, 128), (32768, 32768, 1, 1, 1, 64)):
        assert lib.kaio_b200_attention_paged_int8_scratch(*sizes, C.byref(n)) == 0
        if n.value:
            other = dict(zip(("batch", "tokens", "max_new", "heads", "kv_heads", "head_dim"), sizes))
            bigger = dict(num_pages=1, max_pages=1, q_stride=other["heads"] * other["head_dim"], block_table_len=1 << 20, q_start_len=1 << 20,
                          kv_len_len=1 << 20, k_cache_len=1 << 30, v_cache_len=1 << 30, k_scale_len=1 << 20, v_scale_len=1 << 20,
                          q_len=1 << 40, out_len=1 << 40)
            refused(lib, op, f"scratch too small: need {n.value} f32, got {n.value - 1}", scratch_len=n.value - 1, **other, **bigger)
            refused(lib, op, "scratch pointer is null", null=("scratch",), **other, **bigger, scratch_len=n.value)
            refused(lib, op, "scratch must be 16-byte aligned", odd=("scratch",), **other, **bigger, scratch_len=n.value)


class Recorder:
    """Stands for `kaio_b200.ops`: keeps what it is called with."""

    def attention_paged_int8_scratch(self, *sizes):
        return 0

    def __getattr__(self, name):
        return lambda *args: setattr(self, "last", (name, args))


def holder(heads=4, kv_heads=2, d=64, page=16, pages=3):
    storage = (torch.zeros(pages, kv_heads, page, d, dtype=torch.int8), torch.zeros(pages, kv_heads, page, d, dtype=torch.int8),
               torch.zeros(pages, kv_heads, page // 16), torch.zeros(pages, kv_heads, page // 16))
    rec = Recorder()
    return rec, PagedKvInt8(rec, object(), pages, heads, kv_heads, d, page, storage=storage)


def test_the_holder_passes_parts_of_one_projection():
    """q, k and v as column ranges of one [tokens, 512] matrix: flat buffers that begin at the part, with its stride."""
    rec, cache = holder()
    fused = torch.arange(5 * 512, dtype=torch.float32).half().view(5, 512)
    q, k, v = fused[:, :256], fused[:, 256:384], fused[:, 384:]
    table, start, kv = torch.zeros(2, 3, dtype=torch.int32), torch.zeros(3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    cos = torch.zeros(9, 32)
    cache.append(q, k, v, torch.empty(5, 256).half(), cos, cos, table, start, kv)
    name, a = rec.last
    assert name == "rope_append_kv_int8"
    for got, part in zip(a[1:4], (q, k, v)):
        assert got.dim() == 1 and got.is_contiguous() and got.data_ptr() == part.data_ptr() and got.numel() == 4 * 512 + part.shape[1]
    assert a[14:] == (2, 5, 4, 2, 64, 512, 512, 64, False, 9, 16, 3, 3)
    cache.append(None, k[:1], v[:1], None, None, None, table[:1], start[:2], kv[:1])
    assert rec.last[1][14:] == (1, 1, 4, 2, 64, 0, 128, 0, False, 0, 16, 3, 3)
    cache.attend(q, torch.empty(5, 256).half(), table, start, kv, 3, causal=False)
    assert rec.last[0] == "attention_paged_int8" and rec.last[1][11:] == (2, 5, 3, 4, 2, 64, 512, False, 16, 3, 3)
    cache.gather(k.contiguous(), v.contiguous(), table, start)
    assert rec.last[1][9:] == (2, 5, 2, 64, 16, 3, 3)


def test_the_holder_refuses_what_does_not_fit():
    rec, cache = holder()
    q, k, out = torch.zeros(5, 256).half(), torch.zeros(5, 128).half(), torch.zeros(5, 256).half()
    table, start, kv = torch.zeros(2, 3, dtype=torch.int32), torch.zeros(3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    cos = torch.zeros(9, 32)

    def no(match, *a, **kw):
        with pytest.raises(ValueError, match=match):
            cache.append(*a, **kw)
    no("do not fit", q, k, k, out, cos, cos, table, start[:2], kv)
    no("k: expected a matrix of 128 columns, got shape", q, q, k, out, cos, cos, table, start, kv)
    no("one row stride", q, k, torch.zeros(5, 136).half()[:, :128], out, cos, cos, table, start, kv)
    no("same number of rows", q[:4], k, k, out, cos, cos, table, start, kv)
    no("same number of rows", q, k, k, out[:4], cos, cos, table, start, kv)
    no("same number of rows", q, k, k, None, cos, cos, table, start, kv)
    no("rows are contiguous", q.t().contiguous().t(), k, k, out, cos, cos, table, start, kv)
    no("cos and sin must both be", q, k, k, out, cos, cos[:5], table, start, kv)
    no("cos and sin must both be", q, k, k, out, cos, cos, table, start, kv, rot_dim=32)
    with pytest.raises(ValueError, match="out must have the shape of q"):
        cache.attend(q, out[:4], table, start, kv, 1)
    with pytest.raises(ValueError, match="k_scale: expected shape"):
        PagedKvInt8(rec, object(), 3, 4, 2, 64, 16, storage=(cache.k, cache.v, cache.k_scale[:2], cache.v_scale))
    assert np.all([t.sum().item() == 0 for t in (cache.k, cache.v)])


def test_arrays_read_as_vectors_are_aligned_for_it():
    """An array of f32 or 32-bit words that the kernels read or write as vectors states the alignment, which its element type
    does not give; with less, the address would depend on what the compiler puts beside it."""
    csrc = os.path.join(ROOT, "kaio_b200", "csrc")
    for name in ("attention_paged_decode.cu", "attention_paged_chunk.cu", "kv_append.cu"):
        text = open(os.path.join(csrc, name)).read()
        arrays = {}
        for declaration in re.findall(r"^\s*((?:__shared__ )?(?:alignas\(\d+\) )?(?:volatile )?(?:float|uint32_t|uint8_t|__half)\s[^;()=]*\[[^;]*);", text, re.M):
            for array in re.findall(r"(\w+)\[", declaration):
                arrays[array] = "alignas" in declaration
        for array, _ in re.findall(r"reinterpret_cast<(?:const )?(?:float2|float4|uint2|uint4)\s?\*>\(&?(\w+)([\[)])", text):
            assert arrays.get(array, True), f"{name}: {array} is accessed as a vector without alignas"


def test_a_launch_lets_its_dependents_start_once_it_has_waited():
    """A W4A16 call reads its weights without waiting for the kernel in front; a cache call there must not let it pass the one before."""
    text = open(os.path.join(ROOT, "kaio_b200", "csrc", "kv_cache.cuh")).read()
    body = text[text.index("void kv_begin()"):]
    body = body[:body.index("\n}")]
    assert 0 < body.index("griddepcontrol.wait") < body.index("griddepcontrol.launch_dependents")


def test_a_share_of_units_fits_32_bits(tmp_path, lib):
    """At the most keys that a call is taken with, and one unit more for every (sequence, head); more are refused."""
    run_cpp(tmp_path, r'''
#include <initializer_list>
#include "kv_index.cuh"
using namespace kaio;
int main()
{
    for (uint32_t workers : {32u, 296u, 444u, 480u}) {
        const KvCut c(KV_MOST_KEYS / 128 + (1ull << 27), workers);
        for (uint32_t w = 0; w < workers; ++w)
            if (c.begin(w + 1) - c.begin(w) > 0xffffffffull)
                return 1;
    }
    return 0;
}
''')
    sizes = dict(batch=1 << 15, max_pages=1 << 18, heads=128, kv_heads=128, q_stride=128 * 64, q_len=1 << 20, out_len=1 << 20, k_cache_len=1 << 20,
                 v_cache_len=1 << 20, k_scale_len=1 << 20, v_scale_len=1 << 20, block_table_len=1 << 33, q_start_len=1 << 16, kv_len_len=1 << 16)
    op = "attention_paged_int8"
    refused(lib, op, "batch*max_pages*page_size*kv_heads must be ≤ 2^43 (got 137438953472×128)", **sizes)
    refused(lib, op, "Q buffer too small", **{**sizes, "heads": 64, "kv_heads": 64, "q_len": 1})


def test_no_read_only_loads_in_kernels_that_start_early():
    """The read-only path is for memory that nothing writes while the kernel lives; the kernel in front may still do so while one of
    these is set up."""
    csrc = os.path.join(ROOT, "kaio_b200", "csrc")
    for name in ("attention_paged_decode.cu", "attention_paged_chunk.cu", "kv_append.cu", "kv_cache.cuh"):
        code = re.sub(r"//.*", "", open(os.path.join(csrc, name)).read())
        assert not re.search(r"\.nc\b|__ldg|__restrict__", code), name
