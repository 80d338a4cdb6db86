"""The paged int8 cache on the GPU: appending is compared bit for bit (its f32 steps are part of its definition), attention
with 64 bits within the bound that `kv_reference.attention` derives."""
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

from kaio_b200 import InvalidConfig, ops
from kaio_b200.errors import DeviceTimeout
from kaio_b200.kv_cache import PagedKvInt8
from helpers import device
from kv_reference import Cache

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def cuda(a, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    return t if dtype is None else t.to(dtype)


class Batch:
    """A ragged batch (new tokens, tokens in the cache with them) with its pages in no order, as numpy and on the device."""

    def __init__(self, rng, lens, page, spare_pages=2, spare_rows=0, spare_columns=1):
        self.lens = lens
        need = [-(-kv // page) for _, kv in lens]
        self.pages = sum(need) + spare_pages
        order = rng.permutation(self.pages)
        width = max(need + [0]) + spare_columns
        self.table = np.full((len(lens), max(width, 1)), -1, np.int32)  # what is past the end is not read
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = order[at:at + n]
            at += n
        self.q_start = np.concatenate([[0], np.cumsum([n for n, _ in lens])]).astype(np.int32)
        self.kv_len = np.array([kv for _, kv in lens], np.int32)
        self.rows = int(self.q_start[-1]) + spare_rows
        self.max_new = max(n for n, _ in lens)

    def on_device(self):
        return cuda(self.table), cuda(self.q_start), cuda(self.kv_len)


def on_device(ref, heads):
    return PagedKvInt8(ops, device(), ref.k.shape[0], heads, ref.kv_heads, ref.d, ref.page,
                       storage=tuple(cuda(a) for a in (ref.k, ref.v, ref.ks, ref.vs)))


def tables(positions, rot):
    angle = np.arange(positions)[:, None] * 10000.0 ** (-np.arange(rot // 2) / max(rot // 2, 1))
    return np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)


def same(cache, ref):
    assert np.array_equal(cache.k_scale.cpu().numpy(), ref.ks) and np.array_equal(cache.v_scale.cpu().numpy(), ref.vs)
    assert np.array_equal(cache.k.cpu().numpy(), ref.k) and np.array_equal(cache.v.cpu().numpy(), ref.v)


def append(cache, ref, batch, q, k, v, rot, interleaved, cos, sin):
    """The call and its restatement; rows of no sequence keep what they held."""
    heads = q.shape[1]
    out = torch.full((batch.rows, heads * ref.d), 7.0, dtype=torch.float16, device="cuda")
    cache.append(cuda(q.reshape(batch.rows, -1)), cuda(k.reshape(batch.rows, -1)), cuda(v.reshape(batch.rows, -1)), out,
                 cuda(cos) if rot else None, cuda(sin) if rot else None, *batch.on_device(), interleaved=interleaved)
    want = ref.append(q, k, v, cos, sin, batch.table, batch.q_start, batch.kv_len, rot, interleaved).astype(np.float16)
    want[batch.q_start[-1]:] = 7.0
    assert np.array_equal(out.cpu().numpy().view(np.uint16), want.reshape(batch.rows, -1).view(np.uint16))
    same(cache, ref)


def rows_of(rng, batch, heads, kv_heads, d):
    q, k, v = [rng.standard_normal((batch.rows, n, d)).astype(np.float16) for n in (heads, kv_heads, kv_heads)]
    return q, k, v


LENS = {
    "one": [(1, 1)],
    "steps": [(1, 17), (1, 16), (1, 33), (1, 1), (1, 64), (1, 2)],
    "ragged": [(3, 3), (0, 9), (40, 55), (16, 16), (1, 130), (0, 0), (17, 32), (15, 31)],
    "prompt": [(259, 259)],
    "chunk": [(100, 421)],
    "many": [(i % 3, i % 3 + 5 * (i % 7)) for i in range(70)],
}


@pytest.mark.parametrize("heads,kv_heads,d,page,rot,interleaved", [
    (4, 2, 128, 16, 128, False), (3, 3, 64, 64, 64, False), (2, 1, 128, 32, 32, True), (9, 9, 64, 128, 16, False),
    (8, 1, 128, 256, 64, False), (2, 2, 64, 16, 64, True), (4, 4, 128, 64, 0, False), (12, 4, 128, 64, 112, False)])
@pytest.mark.parametrize("lens", LENS)
def test_append(lens, heads, kv_heads, d, page, rot, interleaved):
    rng = np.random.default_rng(len(lens) * 1000 + heads * d + page)
    batch = Batch(rng, LENS[lens], page, spare_rows=3 if lens == "ragged" else 0)
    ref = Cache(rng, batch.pages, kv_heads, d, page)
    cache = on_device(ref, heads)
    q, k, v = rows_of(rng, batch, heads, kv_heads, d)
    cos, sin = tables(int(batch.kv_len.max()) + 1, rot)
    append(cache, ref, batch, q, k, v, rot, interleaved, cos, sin)
    ops.device_status(device())


def test_append_token_by_token_into_growing_blocks():
    """Forty single tokens, each larger than the last: the scale of a block grows and its tokens move to it."""
    rng = np.random.default_rng(5)
    page, d, heads, kv_heads = 16, 128, 2, 2
    batch = Batch(rng, [(1, 40), (1, 45)], page)
    ref = Cache(rng, batch.pages, kv_heads, d, page)
    cache = on_device(ref, heads)
    cos, sin = tables(64, d)
    for i in range(40):
        batch.kv_len = np.array([i + 1, i + 6], np.int32)
        q, k, v = [x * np.float16(1 + i / 4) for x in rows_of(rng, batch, heads, kv_heads, d)]
        append(cache, ref, batch, q, k, v, d, False, cos, sin)


def test_append_values_that_are_not_numbers():
    """Zeros, the smallest and largest f16, infinities and NaN: each costs its own block and head at most."""
    rng = np.random.default_rng(6)
    page, d = 32, 64
    batch = Batch(rng, [(6, 6), (20, 20), (33, 50), (2, 18)], page)
    ref = Cache(rng, batch.pages, 2, d, page)
    cache = on_device(ref, 2)
    q, k, v = rows_of(rng, batch, 2, 2, d)
    for x in (k, v):
        x[0:6, 0] = 0
        x[0:6, 1] = 6e-8
        x[8, 0, 5], x[9, 0, 6], x[10, 1, 7] = np.inf, -np.inf, np.nan
        x[40, 0, 3], x[41, 1, 4] = 65504, -65504
    cos, sin = tables(64, d)
    append(cache, ref, batch, q, k, v, d, False, cos, sin)
    got_k, got_v = [torch.full((int(batch.kv_len.sum()), 2 * d), 9.0, dtype=torch.float16, device="cuda") for _ in range(2)]
    starts = np.concatenate([[0], np.cumsum(batch.kv_len)]).astype(np.int32)
    cache.gather(got_k, got_v, cuda(batch.table), cuda(starts))
    assert not torch.isnan(got_k).any() and not torch.isnan(got_v).any()
    assert (got_v[0:6, :d] == 0).all() and (got_v[0:6, d:] > 0).all()


def test_append_parts_of_one_projection_in_place():
    rng = np.random.default_rng(8)
    heads, kv_heads, d, page = 4, 2, 64, 16
    batch = Batch(rng, [(5, 30), (1, 7), (18, 18)], page)
    ref = Cache(rng, batch.pages, kv_heads, d, page)
    cache = on_device(ref, heads)
    q, k, v = rows_of(rng, batch, heads, kv_heads, d)
    cos, sin = tables(32, d)
    fused = cuda(np.concatenate([x.reshape(batch.rows, -1) for x in (q, k, v)], 1))
    part = torch.split(fused, [heads * d, kv_heads * d, kv_heads * d], 1)
    out = torch.empty(batch.rows, heads * d, dtype=torch.float16, device="cuda")
    cache.append(*part, out, cuda(cos), cuda(sin), *batch.on_device())
    want = ref.append(q, k, v, cos, sin, batch.table, batch.q_start, batch.kv_len, d, False).astype(np.float16)
    assert np.array_equal(out.cpu().numpy(), want.reshape(batch.rows, -1))
    same(cache, ref)
    # the same tokens again, q rotated in place; what is written is the same
    alone = cuda(q.reshape(batch.rows, -1))
    cache.append(alone, part[1], part[2], alone, cuda(cos), cuda(sin), *batch.on_device())
    assert torch.equal(alone, out)
    ref.append(q, k, v, cos, sin, batch.table, batch.q_start, batch.kv_len, d, False)
    same(cache, ref)
    cache.append(None, part[1], part[2], None, cuda(cos), cuda(sin), *batch.on_device())
    same(cache, ref)


@pytest.mark.parametrize("d,page,kv_heads", [(128, 16, 3), (64, 64, 9), (128, 256, 1)])
def test_gather(d, page, kv_heads):
    rng = np.random.default_rng(d + page)
    batch = Batch(rng, [(0, n) for n in (1, 0, 16, 333, 17, 0, 48)] , page)
    ref = Cache(rng, batch.pages, kv_heads, d, page)
    cache = on_device(ref, kv_heads)
    total = int(batch.kv_len.sum())
    starts = np.concatenate([[0], np.cumsum(batch.kv_len)]).astype(np.int32)
    k, v = [torch.full((total + 2, kv_heads * d), 5.0, dtype=torch.float16, device="cuda") for _ in range(2)]
    cache.gather(k, v, cuda(batch.table), cuda(starts))
    for b in range(len(batch.lens)):
        for got, want in zip((k, v), ref.values(batch.table[b], int(batch.kv_len[b]))):
            # s8 times an f32 scale is rounded to f32 and then to f16
            want = want.reshape(-1, kv_heads * d).astype(np.float32).astype(np.float16)
            assert np.array_equal(got[starts[b]:starts[b + 1]].cpu().numpy(), want)
    assert (k[total:] == 5).all() and (v[total:] == 5).all()


def attend(rng, lens, heads, kv_heads, d, page, causal=True, spare_rows=0, q_scale=1.0, edit=None, max_new=None):
    batch = Batch(rng, lens, page, spare_rows=spare_rows)
    ref = Cache(rng, batch.pages, kv_heads, d, page)
    if edit:
        edit(ref, batch)
    cache = on_device(ref, heads)
    q = (rng.standard_normal((batch.rows, heads, d)) * q_scale).astype(np.float16)
    out = torch.full((batch.rows, heads * d), 3.0, dtype=torch.float16, device="cuda")
    scratch = cache.scratch(len(lens), batch.rows, max_new or batch.max_new)
    if scratch is not None:
        scratch.fill_(float("nan"))  # nothing in it is counted on
    cache.attend(cuda(q.reshape(batch.rows, -1)), out, *batch.on_device(), max_new or batch.max_new, causal=causal, scratch=scratch)
    variant = ops.last_variant()
    want, bound = ref.attend(q, batch.table, batch.q_start, batch.kv_len, causal)
    got = out.cpu().numpy().astype(np.float64).reshape(want.shape)
    end = batch.q_start[-1]
    assert (got[end:] == 3.0).all()
    off = np.abs(got - want)[:end]
    assert (off <= bound[:end]).all(), f"{(off > bound[:end]).sum()} values off, the worst {np.nanmax(off / bound[:end]):.2f} times its bound"
    ops.device_status(device())
    return variant


HEADS = [(4, 4), (8, 2), (8, 1), (9, 3), (16, 1), (5, 1)]


@pytest.mark.parametrize("d,page", [(128, 16), (128, 64), (64, 32), (64, 256)])
@pytest.mark.parametrize("heads,kv_heads", HEADS)
def test_attend_one_token(heads, kv_heads, d, page):
    rng = np.random.default_rng(heads * d + page)
    attend(rng, [(1, n) for n in (1, 2, 15, 16, 17, 31, 32, 33, 257, 1000)], heads, kv_heads, d, page)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("heads,kv_heads", [(4, 4), (8, 1), (6, 2)])
def test_attend_few_tokens(heads, kv_heads, d):
    rng = np.random.default_rng(heads + d)
    for new in (2, 3, 4, 7):
        attend(rng, [(new, new), (new, 70), (1, 33), (0, 12), (new, 300)], heads, kv_heads, d, 16)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("heads,kv_heads", [(2, 2), (8, 1), (6, 2)])
def test_attend_chunks(heads, kv_heads, d, causal):
    rng = np.random.default_rng(heads * 2 + d)
    attend(rng, [(100, 100), (33, 500), (128, 129), (1, 65), (0, 40), (257, 300), (2, 2)], heads, kv_heads, d, 32, causal, spare_rows=5)


@pytest.mark.parametrize("new", [1, 3, 40])
@pytest.mark.parametrize("d", [64, 128])
def test_attend_sees_nothing(d, new):
    """Sequences with fewer tokens in the cache than new ones: the rows in front see no key and are zeros.  Empty caches too."""
    rng = np.random.default_rng(new)
    attend(rng, [(new, new // 2), (new, 0), (new, 20 + new), (0, 0)], 4, 2, d, 16)
    attend(rng, [(new, 0)], 4, 4, d, 16, causal=False)


@pytest.mark.parametrize("new", [1, 2, 50])
@pytest.mark.parametrize("d", [64, 128])
def test_attend_ranges_of_scales(d, new):
    """Scales that differ by many powers of two between blocks, of the values most of all; all-zero blocks at the smallest scale."""
    rng = np.random.default_rng(d + new)

    def edit(ref, batch):
        ref.vs *= np.exp2(rng.integers(-20, 8, ref.vs.shape)).astype(np.float32)
        ref.ks *= np.exp2(rng.integers(-6, 2, ref.ks.shape)).astype(np.float32)
        zero = rng.random(ref.vs.shape) < 0.2
        ref.vs[zero] = 0.0
        ref.v.reshape(*ref.vs.shape, -1)[zero] = 0
    attend(rng, [(new, 400), (new, 90), (new, 1000 + new)], 4, 2, d, 64, edit=edit)


@pytest.mark.parametrize("new", [1, 2, 50])
def test_attend_large_scores(new):
    """Scores spread over hundreds of powers of two: one key takes it all."""
    rng = np.random.default_rng(new)
    attend(rng, [(new, 500), (new, 77)], 4, 2, 128, 16, q_scale=30.0)


@pytest.mark.parametrize("new", [1, 3, 40])
def test_attend_does_not_read_past_the_end(new):
    """Behind a sequence's last token: scales that are NaN or infinite, pages that do not exist."""
    rng = np.random.default_rng(new + 3)

    def edit(ref, batch):
        for b, kv in enumerate(batch.kv_len):
            page, at = batch.table[b][(kv - 1) // ref.page], (kv - 1) % ref.page // 16
            ref.ks[page, :, at + 1:], ref.vs[page, :, at + 1:] = np.nan, np.inf
            ref.k[page, :, (kv - 1) % ref.page + 1:] = -128
    attend(rng, [(new, 130 + new), (new, 41 + new), (new, 64 + new)], 4, 2, 128, 64, edit=edit)


def test_attend_long():
    """One sequence over many splits, against 64 bits; the number of new tokens given too large."""
    rng = np.random.default_rng(11)
    attend(rng, [(1, 20011)], 8, 1, 128, 128)
    attend(rng, [(1, 20011), (2, 5)], 4, 2, 64, 16, max_new=4)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("heads,kv_heads", [(4, 4), (8, 1), (24, 2)])
def test_attend_prompts_and_steps_at_once(heads, kv_heads, d):
    """Sequences with one new token, a few, many and none in one call, over caches long enough to be cut: two kernels share it,
    and rows of no sequence stay as they were."""
    rng = np.random.default_rng(heads * d)
    variant = attend(rng, [(1, 3000), (200, 900), (1, 1), (3, 2500), (0, 70), (70, 70), (1, 1500), (8, 8), (9, 1300)], heads, kv_heads, d, 64,
                     spare_rows=4)
    assert variant == "attention_paged_tcgen05_and_decode"
    # few rows only, more of them in some sequences than in others
    variant = attend(rng, [(1, 4000), (3, 5000), (2, 3000), (1, 20)], 5, 1, d, 64, spare_rows=4)
    assert variant == "attention_paged_decode"


@pytest.mark.parametrize("heads,kv_heads", [(4, 2), (8, 1)])
@pytest.mark.parametrize("d", [64, 128])
def test_attend_with_free_places_in_the_batch(heads, kv_heads, d):
    """A batch of more places than are taken, with gaps of more than a warp between those that are, and caches long enough to be
    cut across the gaps; with eight heads some sequences are the tile kernel's."""
    rng = np.random.default_rng(heads + d)
    free = [(0, 30)]
    for gap in (1, 31, 32, 33, 100, 2000):
        variant = attend(rng, free * gap + [(1, 900), (4, 3000)] + free * gap + [(3, 1), (2, 2000)] + free * 3 + [(4, 40)] + free * gap,
                         heads, kv_heads, d, 64)
        assert variant == ("attention_paged_decode" if heads == 4 else "attention_paged_tcgen05_and_decode")


def test_the_longest_sequence_of_the_tile_kernel():
    """Above 16 rows a sequence of more than 2^25 tokens is left out and reported, before any of its pages is looked up."""
    rng = np.random.default_rng(41)
    batch = Batch(rng, [(40, 70), (40, 90)], 256)
    ref = Cache(rng, batch.pages, 1, 64, 256)
    q = rng.standard_normal((batch.rows, 1, 64)).astype(np.float16)
    want, bound = ref.attend(q, batch.table, batch.q_start, batch.kv_len)
    table = np.full((2, (1 << 17) + 1), -1, np.int32)
    table[:, :batch.table.shape[1]] = batch.table
    out = torch.full((batch.rows, 64), 3.0, dtype=torch.float16, device="cuda")
    on_device(ref, 1).attend(cuda(q.reshape(batch.rows, -1)), out, cuda(table), cuda(batch.q_start),
                             cuda(np.array([70, (1 << 25) + 1], np.int32)), 40)
    with pytest.raises(InvalidConfig, match="kv_len"):
        ops.device_status(device())
    got = out.cpu().numpy().astype(np.float64).reshape(want.shape)
    assert (np.abs(got - want) <= bound)[:40].all() and (got[40:] == 3.0).all()


@pytest.mark.parametrize("heads,kv_heads,new", [(48, 1, 1), (24, 1, 1), (40, 8, 30), (130, 1, 2), (64, 1, 3), (20, 4, 1)])
def test_attend_other_groups(heads, kv_heads, new):
    """Query heads to a key head that no tile is made for: 48, 24, 5, 130."""
    rng = np.random.default_rng(heads + new)
    attend(rng, [(new, 700), (new, 33), (new, new)], heads, kv_heads, 128, 16)


@pytest.mark.parametrize("new", [1, 2, 40])
def test_attend_many_sequences(new):
    """More sequences than a warp has lanes, and than a block sums at once; two of them share all their pages."""
    rng = np.random.default_rng(new)
    attend(rng, [(new if i % 3 else 0, new + (i * 37) % 150) for i in range(70)], 2, 1, 64, 16)
    if new == 1:
        attend(rng, [(i % 2, 1 + (i * 11) % 40) for i in range(1100)], 1, 1, 64, 16)
    batch = Batch(rng, [(new, 100 + new)] * 2, 16)
    batch.table[1] = batch.table[0]
    ref = Cache(rng, batch.pages, 1, 64, 16)
    cache = on_device(ref, 2)
    q = rng.standard_normal((batch.rows, 2, 64)).astype(np.float16)
    out = torch.empty(batch.rows, 128, dtype=torch.float16, device="cuda")
    cache.attend(cuda(q.reshape(batch.rows, -1)), out, *batch.on_device(), new)
    want, bound = ref.attend(q, batch.table, batch.q_start, batch.kv_len)
    assert (np.abs(out.cpu().numpy().astype(np.float64).reshape(want.shape) - want) <= bound).all()


@pytest.mark.parametrize("new", [1, 3, 40])
@pytest.mark.parametrize("d", [64, 128])
def test_attend_rows_that_are_not_numbers(d, new):
    """An infinity or a NaN in a row of q makes that row's output NaN and no other's."""
    rng = np.random.default_rng(d + new)
    heads, kv_heads = 8, 2
    batch = Batch(rng, [(new, 300), (new, 45)], 16)
    ref = Cache(rng, batch.pages, kv_heads, d, 16)
    cache = on_device(ref, heads)
    q = rng.standard_normal((batch.rows, heads, d)).astype(np.float16)
    want, bound = ref.attend(q, batch.table, batch.q_start, batch.kv_len)
    q[0, 1, 3], q[batch.rows - 1, 6, d - 1] = np.nan, np.inf
    out = torch.empty(batch.rows, heads * d, dtype=torch.float16, device="cuda")
    cache.attend(cuda(q.reshape(batch.rows, -1)), out, *batch.on_device(), new)
    got = out.cpu().numpy().astype(np.float64).reshape(want.shape)
    bad = np.zeros(got.shape[:2], bool)
    bad[0, 1] = bad[batch.rows - 1, 6] = True
    assert np.isnan(got[bad]).all()
    assert (np.abs(got - want) <= bound)[~bad].all()


@pytest.mark.parametrize("new", [1, 3, 40])
def test_a_sequence_with_more_new_tokens_than_was_said(new):
    """It is left out and reported; the others are right."""
    rng = np.random.default_rng(new + 1)
    batch = Batch(rng, [(new, 60 + new), (new + 1, 90), (new, 33 + new)], 16)
    ref = Cache(rng, batch.pages, 2, 128, 16)
    cache = on_device(ref, 4)
    q = rng.standard_normal((batch.rows, 4, 128)).astype(np.float16)
    out = torch.full((batch.rows, 512), 3.0, dtype=torch.float16, device="cuda")
    cache.attend(cuda(q.reshape(batch.rows, -1)), out, *batch.on_device(), new)
    with pytest.raises(InvalidConfig, match="more new tokens than max_new"):
        ops.device_status(device())
    want, bound = ref.attend(q, batch.table, batch.q_start, batch.kv_len)
    got = out.cpu().numpy().astype(np.float64).reshape(want.shape)
    for b in (0, 2):
        rows = slice(batch.q_start[b], batch.q_start[b + 1])
        assert (np.abs(got - want)[rows] <= bound[rows]).all()
    assert (got[batch.q_start[1]:batch.q_start[2]] == 3.0).all()


def test_calls_at_once_and_again():
    """Two streams attend at the same time, each with its scratch, eagerly and from captured graphs; every pass gives the same
    bits, whatever ran beside it."""
    rng = np.random.default_rng(21)
    streams = [torch.cuda.Stream() for _ in range(2)]
    work = []
    for lens, heads, kv_heads, new in (([(1, 3000)] * 6, 8, 2, 1), ([(300, 900), (1, 2000)], 8, 2, 300)):
        batch = Batch(rng, lens, 64)
        ref = Cache(rng, batch.pages, kv_heads, 128, 64)
        cache = on_device(ref, heads)
        q = rng.standard_normal((batch.rows, heads, 128)).astype(np.float16)
        out = torch.empty(batch.rows, heads * 128, dtype=torch.float16, device="cuda")
        args = (cuda(q.reshape(batch.rows, -1)), out, *batch.on_device(), new)
        cache.attend(*args)
        want, bound = ref.attend(q, batch.table, batch.q_start, batch.kv_len)
        assert (np.abs(out.cpu().numpy().astype(np.float64).reshape(want.shape) - want) <= bound).all()
        work.append((cache, args, out, out.clone(), cache.scratch(len(lens), batch.rows, new)))
    torch.cuda.synchronize()
    graphs = []
    for stream, (cache, args, out, _, scratch) in zip(streams, work):
        cache.device = ops.KaioDevice(0, stream)
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=stream):
            cache.attend(*args, scratch=scratch)
    for i in range(20):
        for _, _, out, _, _ in work:
            out.zero_()
        torch.cuda.synchronize()
        for stream, graph, (cache, args, _, _, scratch) in zip(streams, graphs, work):
            with torch.cuda.stream(stream):
                graph.replay() if i % 2 else cache.attend(*args, scratch=scratch if i % 4 else None)
        torch.cuda.synchronize()
        for _, _, out, first, _ in work:
            assert torch.equal(out, first)
    ops.device_status(device())


def test_calls_right_behind_one_another():
    """Append, attend and read back over steps, prompts and both, each call set up while the one in front of it runs: the same
    bits as with a pause after each, eagerly and from a graph."""
    rng = np.random.default_rng(22)
    heads, kv_heads, d, page, width = 8, 2, 128, 16, 32
    ref = Cache(rng, 4 * width, kv_heads, d, page)
    table = cuda(rng.permutation(4 * width).astype(np.int32).reshape(4, width))
    cos, sin = (cuda(x) for x in tables(width * page, d))
    steps, kv = [], np.zeros(4, np.int32)
    for new in ([60, 33, 5, 1], [1, 1, 1, 1], [1, 1, 1, 1], [1, 90, 0, 3], [4, 2, 4, 1], [40, 40, 40, 40], [1, 0, 1, 1], [3, 3, 3, 3],
                [16, 12, 16, 16], [1, 1, 1, 1]):
        kv = kv + np.array(new, np.int32)
        rows = sum(new)
        q, k, v = (cuda(rng.standard_normal((rows, n * d)).astype(np.float16)) for n in (heads, kv_heads, kv_heads))
        steps.append((q, k, v, torch.empty_like(q), torch.empty_like(q), cuda(np.concatenate([[0], np.cumsum(new)]).astype(np.int32)), cuda(kv),
                      cuda(np.concatenate([[0], np.cumsum(kv)]).astype(np.int32)),
                      [torch.empty(int(kv.sum()), kv_heads * d, dtype=torch.float16, device="cuda") for _ in range(2)], max(new)))
    cache = on_device(ref, heads)
    first = [x.clone() for x in (cache.k, cache.v, cache.k_scale, cache.v_scale)]
    scratch = torch.empty(max((cache.scratch(4, s[0].shape[0], s[-1]).numel() for s in steps)), device="cuda")
    pause = torch.cuda.synchronize

    def run(after):
        for x, y in zip((cache.k, cache.v, cache.k_scale, cache.v_scale), first):
            x.copy_(y)
        for q, k, v, turned, out, start, kv_len, kv_start, back, max_new in steps:
            cache.append(q, k, v, turned, cos, sin, table, start, kv_len)
            after()
            cache.attend(turned, out, table, start, kv_len, max_new, scratch=scratch)
            after()
            cache.gather(*back, table, kv_start)
            after()

    def results():
        pause()
        got = [x.clone() for s in steps for x in (s[3], s[4], *s[8])] + [cache.k.clone(), cache.v.clone()]
        for s in steps:
            for x in (s[3], s[4], *s[8]):
                x.zero_()
        pause()
        return got
    run(pause)
    want = results()
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    cache.device = ops.KaioDevice(0, stream)
    with torch.cuda.graph(graph, stream=stream):
        run(lambda: None)
    for i in range(10):
        with torch.cuda.stream(stream):
            run(lambda: None) if i % 2 else graph.replay()
        for got, expect in zip(results(), want):
            assert torch.equal(got, expect)
    ops.device_status(device())


def test_pages_past_two_to_the_31_values():
    """A cache of 2.2 GB each of keys and values whose sequences lie in its last pages, against the same pages at the front of a
    small one."""
    rng = np.random.default_rng(31)
    heads, kv_heads, d, page, pages = 16, 8, 128, 64, 33000
    batch = Batch(rng, [(1, 200), (40, 77), (1, 64)], page)
    ref = Cache(rng, batch.pages, kv_heads, d, page)
    storage = (torch.zeros(pages, kv_heads, page, d, dtype=torch.int8, device="cuda"), torch.zeros(pages, kv_heads, page, d, dtype=torch.int8, device="cuda"),
               torch.zeros(pages, kv_heads, page // 16, device="cuda"), torch.zeros(pages, kv_heads, page // 16, device="cuda"))
    first = pages - batch.pages
    for big, small in zip(storage, (ref.k, ref.v, ref.ks, ref.vs)):
        big[first:] = cuda(small)
    cache = PagedKvInt8(ops, device(), pages, heads, kv_heads, d, page, storage=storage)
    table, start, kv = batch.on_device()
    table = torch.where(table >= 0, table + first, table)
    cos, sin = tables(256, d)
    q, k, v = rows_of(rng, batch, heads, kv_heads, d)
    turned = torch.empty(batch.rows, heads * d, dtype=torch.float16, device="cuda")
    cache.append(*[cuda(x.reshape(batch.rows, -1)) for x in (q, k, v)], turned, cuda(cos), cuda(sin), table, start, kv)
    want_q = ref.append(q, k, v, cos, sin, batch.table, batch.q_start, batch.kv_len, d, False).astype(np.float16)
    for big, small in zip(storage, (ref.k, ref.v, ref.ks, ref.vs)):
        assert np.array_equal(big[first:].cpu().numpy(), small) and not big[:first].any()
    out = torch.empty(batch.rows, heads * d, dtype=torch.float16, device="cuda")
    for max_new in (40, 64):
        cache.attend(turned, out, table, start, kv, max_new)
        want, bound = ref.attend(want_q, batch.table, batch.q_start, batch.kv_len)
        assert (np.abs(out.cpu().numpy().astype(np.float64).reshape(want.shape) - want) <= bound).all()
    got_k, got_v = [torch.empty(int(batch.kv_len.sum()), kv_heads * d, dtype=torch.float16, device="cuda") for _ in range(2)]
    starts = np.concatenate([[0], np.cumsum(batch.kv_len)]).astype(np.int32)
    cache.gather(got_k, got_v, table, cuda(starts))
    for b in range(3):
        want_k, _ = ref.values(batch.table[b], int(batch.kv_len[b]))
        assert np.array_equal(got_k[starts[b]:starts[b + 1]].cpu().numpy(), want_k.reshape(-1, kv_heads * d).astype(np.float32).astype(np.float16))
    ops.device_status(device())


def test_bad_numbers_are_left_out_and_reported():
    """Pages, lengths and row starts that lead outside their buffers: the sequences beside them are right, and the status
    names what was found."""
    rng = np.random.default_rng(12)
    heads, kv_heads, d, page = 4, 2, 128, 16
    for new in (1, 3, 40):
        batch = Batch(rng, [(new, 50 + new)] * 3, page)
        ref = Cache(rng, batch.pages, kv_heads, d, page)
        q, k, v = rows_of(rng, batch, heads, kv_heads, d)
        want, bound = ref.attend(q, batch.table, batch.q_start, batch.kv_len)
        edits = [("table", (1, 0), batch.pages, "block_table"), ("table", (1, 2), -5, "block_table"),
                 ("kv_len", (1,), 1 << 30, "kv_len"), ("kv_len", (1,), -4, "kv_len")]
        edits += [("q_start", (2,), 4096, "q_start"), ("q_start", (1,), -7, "q_start")]
        for name, at, value, text in edits:
            arrays = {n: getattr(batch, n).copy() for n in ("table", "q_start", "kv_len")}
            arrays[name][at] = value
            cache = on_device(ref, heads)
            out = torch.zeros(batch.rows, heads * d, dtype=torch.float16, device="cuda")
            cache.attend(cuda(q.reshape(batch.rows, -1)), out, *[cuda(arrays[n]) for n in ("table", "q_start", "kv_len")], new)
            with pytest.raises(InvalidConfig, match=text):
                ops.device_status(device())
            got = out.cpu().numpy().astype(np.float64).reshape(want.shape)
            for b in (0, 2) if name != "q_start" else (0,) if at == (2,) else (2,):
                rows = slice(batch.q_start[b], batch.q_start[b + 1])
                assert (np.abs(got - want)[rows] <= bound[rows]).all(), (name, b)
            assert np.isfinite(got).all()
        # appending: a page outside the cache and positions outside the rotation table
        cos, sin = tables(50 + new, d)
        for name, at, value, text, positions in (("table", (1, 3), 99999, "block_table", 50 + new), ("kv_len", (1,), 51 + new, "kv_len", 50 + new),
                                                 ("kv_len", (1,), new - 1, "kv_len", 50 + new), ("q_start", (3,), 4096, "q_start", 50 + new)):
            arrays = {n: getattr(batch, n).copy() for n in ("table", "q_start", "kv_len")}
            arrays[name][at] = value
            cache, plain = on_device(ref, heads), ref.copy()
            out = torch.zeros(batch.rows, heads * d, dtype=torch.float16, device="cuda")
            cache.append(*[cuda(x.reshape(batch.rows, -1)) for x in (q, k, v)], out, cuda(cos), cuda(sin),
                         *[cuda(arrays[n]) for n in ("table", "q_start", "kv_len")])
            with pytest.raises(InvalidConfig, match=text):
                ops.device_status(device())
            plain.append(q, k, v, cos, sin, batch.table, batch.q_start, batch.kv_len, d, False)
            for b in ((0, 1) if name == "q_start" else (0, 2)):
                pages = batch.table[b][:-(-int(batch.kv_len[b]) // page)].astype(np.int64)
                assert np.array_equal(cache.k.cpu().numpy()[pages], plain.k[pages])
                assert np.array_equal(cache.v.cpu().numpy()[pages], plain.v[pages])
    ops.device_status(device())


def test_steps_as_a_serving_program_makes_them():
    """A prompt and six steps of three sequences: append, attend and read back, each step from the last one's cache; the steps
    from one captured graph on a stream of its own, whose lengths change between replays."""
    rng = np.random.default_rng(13)
    heads, kv_heads, d, page = 8, 2, 128, 16
    lens = [(37, 37), (5, 5), (64, 64)]
    batch = Batch(rng, [(n, n + 8) for n, _ in lens], page, spare_columns=0)
    ref = Cache(rng, batch.pages, kv_heads, d, page)
    cache = on_device(ref, heads)
    cos, sin = tables(128, d)
    prompt = Batch(rng, lens, page)
    prompt.table, prompt.pages = batch.table, batch.pages
    q, k, v = rows_of(rng, prompt, heads, kv_heads, d)
    append(cache, ref, prompt, q, k, v, d, False, cos, sin)
    out = torch.empty(prompt.rows, heads * d, dtype=torch.float16, device="cuda")
    turned = ref.append(q, k, v, cos, sin, prompt.table, prompt.q_start, prompt.kv_len, d, False).astype(np.float16)
    cache.attend(cuda(turned.reshape(prompt.rows, -1)), out, *prompt.on_device(), 64)
    want, bound = ref.attend(turned, prompt.table, prompt.q_start, prompt.kv_len)
    assert (np.abs(out.cpu().numpy().astype(np.float64).reshape(want.shape) - want) <= bound).all()

    stream = torch.cuda.Stream()
    cache.device = ops.KaioDevice(0, stream)
    start, kv = np.arange(4, dtype=np.int32), np.array([n for n, _ in lens], np.int32)
    table_d, start_d, kv_d, cos_d, sin_d = cuda(batch.table), cuda(start), cuda(kv), cuda(cos), cuda(sin)
    qkv = torch.zeros(3, (heads + 2 * kv_heads) * d, dtype=torch.float16, device="cuda")
    part = torch.split(qkv, [heads * d, kv_heads * d, kv_heads * d], 1)
    turned_d, out = [torch.zeros(3, heads * d, dtype=torch.float16, device="cuda") for _ in range(2)]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        kv_d += 1
        cache.append(*part, turned_d, cos_d, sin_d, table_d, start_d, kv_d)
        cache.attend(turned_d, out, table_d, start_d, kv_d, 1)
    for _ in range(6):
        x = rng.standard_normal((3, qkv.shape[1])).astype(np.float16)
        qkv.copy_(cuda(x))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        kv = kv + 1
        q, k, v = [p.reshape(3, -1, d) for p in np.split(x, [heads * d, (heads + kv_heads) * d], 1)]
        turned = ref.append(q, k, v, cos, sin, batch.table, start, kv, d, False).astype(np.float16)
        same(cache, ref)
        want, bound = ref.attend(turned, batch.table, start, kv)
        assert (np.abs(out.cpu().numpy().astype(np.float64).reshape(want.shape) - want) <= bound).all()
    ops.device_status(device())


def a_page_that_is_not_there():
    """Attention of one token whose page lies outside the cache: left out and reported."""
    rng = np.random.default_rng(40)
    batch = Batch(rng, [(1, 20)], 16)
    ref = Cache(rng, batch.pages, 1, 64, 16)
    batch.table[0, 0] = batch.pages
    q, out = [torch.zeros(1, 64, dtype=torch.float16, device="cuda") for _ in range(2)]
    on_device(ref, 1).attend(q, out, *batch.on_device(), 1)


@pytest.mark.parametrize("first", ["index", "wait"])
def test_a_wait_that_gave_up_is_reported_beside_a_bad_index(first):
    for what in ("index", "wait") if first == "index" else ("wait", "index"):
        a_page_that_is_not_there() if what == "index" else ops.selftest_bounded_wait(device(), 5)
    with pytest.raises(DeviceTimeout, match="code 1"):
        ops.device_status(device())
    with pytest.raises(InvalidConfig, match="block_table"):
        ops.device_status(device())
    assert ops.device_status(device()) == [0, 0, 0, 0]


def test_a_cache_call_between_a_writer_of_weights_and_their_reader():
    """Scales that a read back writes, an append behind it, and a W4A16 call of one row that reads them without waiting for the kernel
    directly in front: what was in front of the append is done when the append lets its dependents start."""
    rng = np.random.default_rng(41)
    k_dim, n, kv_heads, d, page, tokens = 1024, 4096, 8, 128, 64, 8192
    pages = tokens // page + 1
    storage = (torch.zeros(pages, kv_heads, page, d, dtype=torch.int8, device="cuda"), torch.zeros(pages, kv_heads, page, d, dtype=torch.int8, device="cuda"),
               torch.ones(pages, kv_heads, page // 16, device="cuda"), torch.ones(pages, kv_heads, page // 16, device="cuda"))
    cache = PagedKvInt8(ops, device(), pages, kv_heads, kv_heads, d, page, storage=storage)
    x = cuda(rng.standard_normal(k_dim).astype(np.float16))
    packed = cuda(rng.integers(-2 ** 31, 2 ** 31, k_dim // 8 * n).astype(np.int32))
    back = [torch.zeros(tokens, kv_heads * d, dtype=torch.float16, device="cuda") for _ in range(2)]
    scales = back[0].view(-1)[-(k_dim // 128) * n:]  # what the last blocks write
    table = cuda(np.arange(pages - 1, dtype=np.int32)[None])
    own, start, one, kv = (cuda(np.array(a, np.int32)) for a in ([[pages - 1]], [0, tokens], [0, 1], [1]))
    new = torch.ones(1, kv_heads * d, dtype=torch.float16, device="cuda")
    c, want = [torch.zeros(n, dtype=torch.float32, device="cuda") for _ in range(2)]
    ops.matmul_int4(device(), x, packed, scales, c, 1, n, k_dim, 128)
    for i in range(30):
        cache.k.copy_(torch.randint(1, 128, cache.k.shape, dtype=torch.int8, device="cuda"))
        torch.cuda.synchronize()
        cache.gather(*back, table, start)
        cache.append(None, new, new, None, None, None, own, one, kv)
        ops.matmul_int4(device(), x, packed, scales, c, 1, n, k_dim, 128)
        torch.cuda.synchronize()
        ops.matmul_int4(device(), x, packed, scales, want, 1, n, k_dim, 128)
        torch.cuda.synchronize()
        assert torch.equal(c, want) and want.abs().max() > 0
    ops.device_status(device())


EDGES = r"""
import sys, torch
from cuda.bindings import runtime as rt
sys.path.insert(0, sys.argv[1])
from kaio_b200 import ops
from kaio_b200.kv_cache import PagedKvInt8
dev = ops.KaioDevice(0)
cache = PagedKvInt8(ops, dev, 8, 8, 1, 64, 16)
q, k, v, turned, out = [torch.ones(40, n, dtype=torch.float16, device="cuda") for n in (512, 64, 64, 512, 512)]
table, start, kv = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([[1, 2], [3, 4]], [0, 39, 40], [39 - 16, 1])]
back = [torch.empty(24, 64, dtype=torch.float16, device="cuda") for _ in range(2)]
ends = torch.tensor([0, 23, 24], dtype=torch.int32, device="cuda")
scratch = cache.scratch(2, 40, 40)


def calls():
    cache.append(q, k, v, turned, None, None, table, start, kv)
    cache.attend(turned, out, table, start, kv, 40, scratch=scratch)
    cache.attend(turned[:1], out[:1], table[:1], start[:2], kv[:1], 1, scratch=scratch)
    cache.gather(*back, table, ends)


calls()
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph(keep_graph=True)
with torch.cuda.graph(graph):
    calls()
raw = rt.cudaGraph_t(graph.raw_cuda_graph())
count = rt.cudaGraphGetEdges_v2(raw)[-1]
err, _, _, data, count = rt.cudaGraphGetEdges_v2(raw, count)
assert err == rt.cudaError_t.cudaSuccess
print("edges", len(data), "programmatic", sum(int(e.type) == 1 for e in data))
"""


@pytest.mark.parametrize("value", ["0", None])
def test_plain_serialisation_on_request(value):
    """KAIO_B200_PDL=0: no launch of the cache's calls starts before the one in front is done."""
    env = {k: v for k, v in os.environ.items() if k != "KAIO_B200_PDL"}
    if value is not None:
        env["KAIO_B200_PDL"] = value
    r = subprocess.run([sys.executable, "-c", EDGES, ROOT], capture_output=True, text=True, timeout=300, env=env)
    assert r.returncode == 0, r.stderr[-2000:]
    edges, programmatic = [int(x) for x in r.stdout.split()[1::2]]
    assert edges >= 5 and (programmatic == 0 if value == "0" else programmatic >= 4), r.stdout


def test_a_long_sequence_beside_prompts():
    """In a call that both kernels share, a sequence of more than 2^25 tokens with one new one is the few-row kernel's: computed, and
    not reported as left out.  All its table entries name one page, so its softmax is that page's."""
    rng = np.random.default_rng(33)
    d, page, heads = 64, 256, 2
    n_pages = (1 << 25) // page + 3
    batch = Batch(rng, [(40, 70), (1, 1)], page)
    ref = Cache(rng, batch.pages, 1, d, page)
    q = rng.standard_normal((batch.rows, heads, d)).astype(np.float16)
    table = np.full((2, n_pages), batch.table[1, 0], np.int32)
    table[0, 0] = batch.table[0, 0]
    out = torch.full((batch.rows, heads * d), 3.0, dtype=torch.float16, device="cuda")
    on_device(ref, heads).attend(cuda(q.reshape(batch.rows, -1)), out, cuda(table), cuda(batch.q_start),
                                 cuda(np.array([70, n_pages * page], np.int32)), 40)
    assert ops.last_variant() == "attention_paged_tcgen05_and_decode"
    want, bound = ref.attend(q, batch.table, batch.q_start, np.array([70, page], np.int32))
    # the sums run over 2^17 times the keys: parts of at most 2^25 / 444 keys each in f32
    bound = bound + np.abs(want) * 2.0 ** -24 * (1 << 17)
    got = out.cpu().numpy().astype(np.float64).reshape(want.shape)
    assert (np.abs(got - want) <= bound).all()
    assert ops.device_status(device()) == [0, 0, 0, 0]


@pytest.mark.parametrize("above", [11.0, 13.0, 15.0])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("heads,kv_heads,new,sequences", [(1, 1, 1, 512), (12, 1, 1, 512), (2, 2, 300, 2), (4, 1, 20, 40)])
def test_attend_behind_a_dominant_first_key(heads, kv_heads, new, sequences, d, above):
    """Flat scores behind a first key that is `above` them in the exponent and whose values are zeros, as trained models
    have it: the others' P stay out of f16's subnormal range.  The bound of `kv_reference.attention` counts 2^-25 for each P below
    the normal range where the largest is at least 1; here it is at least 2^7."""
    rng = np.random.default_rng(int(above) + new + d)
    batch = Batch(rng, [(new, 2000 + new + 7 * (i % 3)) for i in range(2)], 64)
    ref = Cache(rng, batch.pages, kv_heads, d, 64)
    q = np.ones((batch.rows, heads, d), np.float16)
    ref.k[:] = 0
    ref.v[:] = rng.integers(20, 128, ref.v.shape)
    for b in range(2):
        page = batch.table[b, 0]
        ref.k[page, :, 0], ref.v[page, :, 0] = 100, 0
        ref.ks[page, :, 0] = above * np.sqrt(d) / (100 * d)
    want, bound = ref.attend(q, batch.table, batch.q_start, batch.kv_len)
    for b, (n, kv) in enumerate(batch.lens):
        # what `attend` counted for it, with the largest scale of the sequence's pages and the head, less 1 part in 2^7
        keys, vs = kv - n + 1 + np.arange(n), ref.vs[batch.table[b][:-(-kv // 64)].astype(np.int64)].max((0, 2))
        counted = keys[:, None] * 2.0 ** -25 * 127 * vs.repeat(heads // kv_heads)
        bound[b * n:(b + 1) * n] -= counted[..., None] * (1 - 2.0 ** -7)
    cache = on_device(ref, heads)
    # the two sequences again and again: enough of them that none is cut
    table, start, kv = np.tile(batch.table, (sequences // 2, 1)), np.arange(sequences + 1, dtype=np.int32) * new, np.tile(batch.kv_len, sequences // 2)
    out = torch.empty(sequences * new, heads * d, dtype=torch.float16, device="cuda")
    cache.attend(torch.ones_like(out), out, cuda(table), cuda(start), cuda(kv), new)
    got = out.cpu().numpy().astype(np.float64).reshape(sequences // 2, *want.shape)
    off = np.abs(got - want)
    assert (off <= bound).all(), f"{(off > bound).sum()} of {off.size} values off, the worst {(off / bound).max():.2f} times its bound, {(off / np.maximum(want, 1e-9)).max():.1e} of the value"
    ops.device_status(device())


@pytest.mark.parametrize("new", [1, 3, 40, 300])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("size", [1.0, 50.0, 3000.0])
def test_attend_scores_past_two_to_the_24(size, d, new):
    """Keys as an infinity in their block leaves them and large queries: scores whose f32 step is more than one, of either sign.  One key
    has all the weight where it is ahead by more than their rounding, and its values are the output."""
    rng = np.random.default_rng(int(size) + d + new)
    heads, kv_heads = 4, 2
    batch = Batch(rng, [(new, 500 + new), (new, 77 + new)], 16)
    ref = Cache(rng, batch.pages, kv_heads, d, 16)
    ref.ks[:] = np.float32(131008.0) / np.float32(127.0) * (1 + 0.3 * rng.random(ref.ks.shape).astype(np.float32))
    ref.vs *= np.exp2(rng.integers(-6, 3, ref.vs.shape)).astype(np.float32)
    q = (rng.standard_normal((batch.rows, heads, d)) * size).astype(np.float16)
    out = torch.empty(batch.rows, heads * d, dtype=torch.float16, device="cuda")
    on_device(ref, heads).attend(cuda(q.reshape(batch.rows, -1)), out, *batch.on_device(), new)
    got = out.cpu().numpy().astype(np.float64).reshape(q.shape)
    assert np.isfinite(got).all()
    alone = 0
    for b in range(2):
        k, v = ref.values(batch.table[b], int(batch.kv_len[b]))
        for i in range(new):
            n = int(batch.kv_len[b]) - new + i + 1
            for h in range(heads):
                row = q[batch.q_start[b] + i, h].astype(np.float64)
                x = k[:n, h // 2] @ row / np.sqrt(d)
                order = np.argsort(x)
                # f32 sums of d products, scaled and added to once more: (d + 4) 2^-24 of the sum of their sizes
                if x[order[-1]] - x[order[-2]] > 40 + 2 * (d + 4) * 2.0 ** -24 * np.abs(row).sum() * np.abs(k[:n, h // 2]).max() / np.sqrt(d):
                    alone += 1
                    top = v[order[-1], h // 2]
                    assert (np.abs(got[batch.q_start[b] + i, h] - top) <= 2.0 ** -10 * np.abs(top) + 2.0 ** -24).all()
    assert alone > 0


FIRST_CALL = r"""
import sys, torch
sys.path.insert(0, sys.argv[1])
from kaio_b200 import ops
from kaio_b200.kv_cache import PagedKvInt8
cache = PagedKvInt8(ops, ops.KaioDevice(0), 2, 2, 1, 64, 16)
q, k, v, turned, out = [torch.ones(1, n, dtype=torch.float16, device="cuda") for n in (128, 64, 64, 128, 128)]
table, start, kv = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([[1]], [0, 1], [1])]
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    cache.append(q, k, v, turned, None, None, table, start, kv)
    cache.attend(turned, out, table, start, kv, 1)
graph.replay()
torch.cuda.synchronize()
assert (out == 1).all(), out
assert ops.device_status(ops.KaioDevice(0)) == [0, 0, 0, 0]
"""


def test_the_first_call_of_a_process_may_be_captured():
    r = subprocess.run([sys.executable, "-c", FIRST_CALL, ROOT], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]


def compare(got, want, bound, rows=slice(None)):
    off = np.abs(got.cpu().numpy().astype(np.float64).reshape(want.shape) - want)[rows]
    assert (off <= bound[rows]).all(), f"{(off > bound[rows]).sum()} values off, the worst {np.nanmax(off / bound[rows]):.2f} times its bound"


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("heads,kv_heads,lens", [
    # Q by TMA: 256-row items, and what is left of a sequence's rows in items of one tile
    (32, 32, [(300, 300), (520, 700), (129, 129), (256, 260), (90, 1000), (700, 700), (385, 500), (30, 31)]),
    # Q by rows: 24 heads to a key head
    (192, 8, [(100, 140), (33, 400), (8, 8), (64, 64), (51, 300), (16, 2000), (20, 20), (128, 130)]),
    # no sequence has more rows than a tile
    (32, 8, [(5 + 9 * (i % 4), 200 + 37 * (i % 11) + 5 + 9 * (i % 4)) for i in range(64)])])
def test_attend_several_items_for_every_block_that_stays(heads, kv_heads, lens, d):
    """More items with rows than two for each SM, two tiles' and one tile's after each other, so that barriers, rings and tensor
    memory are used on from item to item."""
    rng = np.random.default_rng(heads + d)
    group = heads // kv_heads
    items = sum(-(-n * group // 256) for n, _ in lens) * kv_heads
    assert items > 2 * torch.cuda.get_device_properties(0).multi_processor_count
    for causal in (True, False):
        assert "tcgen05" in attend(rng, lens, heads, kv_heads, d, 64, causal)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("heads,kv_heads,lens,causal", [
    (8, 2, [(1, 500), (1, 30)], True), (8, 2, [(3, 500), (2, 30)], False), (4, 1, [(3, 700), (4, 4)], False),
    (8, 1, [(90, 300), (1, 900), (40, 40)], True), (6, 2, [(90, 300), (45, 70)], False), (24, 1, [(9, 100), (20, 30)], True)])
def test_attend_part_of_a_wider_matrix(heads, kv_heads, lens, causal, d):
    """q as a column range of the projection's output: its rows are longer than its heads.  The rest is NaN."""
    rng = np.random.default_rng(heads + len(lens) + d)
    batch = Batch(rng, lens, 32, spare_rows=2)
    ref = Cache(rng, batch.pages, kv_heads, d, 32)
    q = rng.standard_normal((batch.rows, heads, d)).astype(np.float16)
    wide = torch.full((batch.rows, heads * d + 72), float("nan"), dtype=torch.float16, device="cuda")
    part = wide[:, 24:24 + heads * d]
    part.copy_(cuda(q.reshape(batch.rows, -1)))
    out = torch.full((batch.rows, heads * d), 3.0, dtype=torch.float16, device="cuda")
    on_device(ref, heads).attend(part, out, *batch.on_device(), batch.max_new, causal=causal)
    want, bound = ref.attend(q, batch.table, batch.q_start, batch.kv_len, causal)
    compare(out, want, bound, slice(0, batch.q_start[-1]))
    assert (out[batch.q_start[-1]:] == 3.0).all()
    ops.device_status(device())


@pytest.mark.parametrize("max_new", [1, 3, 300])
def test_calls_whose_rows_belong_to_no_sequence(max_new):
    """A captured step whose places are all free: nothing is written."""
    rng = np.random.default_rng(50)
    for places in (1, 40):
        batch = Batch(rng, [(0, 20)] * places, 16, spare_rows=places)
        batch.max_new = max_new
        ref = Cache(rng, batch.pages, 2, 64, 16)
        cache = on_device(ref, 8)
        q, k, v = rows_of(rng, batch, 8, 2, 64)
        append(cache, ref, batch, q, k, v, 64, False, *tables(64, 64))
        out = torch.full((batch.rows, 512), 3.0, dtype=torch.float16, device="cuda")
        cache.attend(cuda(q.reshape(batch.rows, -1)), out, *batch.on_device(), max_new)
        assert (out == 3.0).all()
        back = [torch.full((2, 128), 5.0, dtype=torch.float16, device="cuda") for _ in range(2)]
        cache.gather(*back, *batch.on_device()[:2])
        assert all((x == 5.0).all() for x in back)
    ops.device_status(device())


def test_the_largest_batch():
    """32768 sequences in each call, a few of them with rows, one with many."""
    rng = np.random.default_rng(51)
    lens = [(1, 1 + i % 30) if i % 1000 == 7 else (0, 0) for i in range(32768)]
    lens[0], lens[-1] = (1, 700), (2, 40)
    batch = Batch(rng, lens, 16)
    ref = Cache(rng, batch.pages, 1, 64, 16)
    cache = on_device(ref, 2)
    q, k, v = rows_of(rng, batch, 2, 1, 64)
    append(cache, ref, batch, q, k, v, 64, False, *tables(1024, 64))
    want, bound = ref.attend(q, batch.table, batch.q_start, batch.kv_len)
    for max_new in (2, 100):
        out = torch.empty(batch.rows, 128, dtype=torch.float16, device="cuda")
        cache.attend(cuda(q.reshape(batch.rows, -1)), out, *batch.on_device(), max_new)
        compare(out, want, bound)
    starts = np.concatenate([[0], np.cumsum(batch.kv_len)]).astype(np.int32)
    got = [torch.empty(int(starts[-1]), 64, dtype=torch.float16, device="cuda") for _ in range(2)]
    cache.gather(*got, cuda(batch.table), cuda(starts))
    for x, y in zip(got, ref.values(batch.table[-1], 40)):
        assert np.array_equal(x[-40:].cpu().numpy(), y[:, 0].astype(np.float32).astype(np.float16))
    ops.device_status(device())


@pytest.mark.parametrize("heads,kv_heads", [(32768, 1), (32768, 4096), (4096, 4096)])
def test_the_most_heads(heads, kv_heads):
    """All the heads that a call takes, of one token and of three."""
    rng = np.random.default_rng(52)
    d, page = 64, 16
    for lens in ([(1, 20)], [(3, 20), (1, 5)]):
        batch = Batch(rng, lens, page)
        ref = Cache(rng, batch.pages, kv_heads, d, page)
        cache = on_device(ref, heads)
        q, k, v = rows_of(rng, batch, heads, kv_heads, d)
        append(cache, ref, batch, q, k, v, d, False, *tables(64, d))
        out = torch.empty(batch.rows, heads * d, dtype=torch.float16, device="cuda")
        cache.attend(cuda(q.reshape(batch.rows, -1)), out, *batch.on_device(), batch.max_new)
        want, bound = ref.attend(q, batch.table, batch.q_start, batch.kv_len)
        compare(out, want, bound)
    ops.device_status(device())


def test_calls_captured_on_forked_streams():
    """A graph whose calls follow kernels of another stream: prompts and steps append and attend on streams of their own behind one
    copy, and a read back behind both."""
    rng = np.random.default_rng(53)
    heads, kv_heads, d, page = 8, 2, 64, 16
    batch = Batch(rng, [(70, 70), (1, 300), (1, 40)], page)
    ref = Cache(rng, batch.pages, kv_heads, d, page)
    cache = on_device(ref, heads)
    q, k, v = rows_of(rng, batch, heads, kv_heads, d)
    cos, sin = tables(512, d)
    table, start, kv = batch.on_device()
    cos_d, sin_d = cuda(cos), cuda(sin)
    source = [cuda(x.reshape(batch.rows, -1)) for x in (q, k, v)]
    given = [torch.zeros_like(x) for x in source]
    turned, out = torch.zeros_like(source[0]), torch.zeros_like(source[0])
    starts = cuda(np.concatenate([[0], np.cumsum(batch.kv_len)]).astype(np.int32))
    back = [torch.zeros(int(batch.kv_len.sum()), kv_heads * d, dtype=torch.float16, device="cuda") for _ in range(2)]
    parts = [(slice(0, 1), slice(0, 70), 70), (slice(1, 3), slice(70, 72), 1)]
    starts_of = [cuda(np.array(s, np.int32)) for s in ([0, 70], [0, 1, 2])]
    first = [x.clone() for x in (cache.k, cache.v, cache.k_scale, cache.v_scale)]
    scratch = [cache.scratch(s.stop - s.start, r.stop - r.start, m) for s, r, m in parts]
    side = [torch.cuda.Stream() for _ in range(2)]

    def calls():
        main = torch.cuda.current_stream()
        for x, y in zip((*given, cache.k, cache.v, cache.k_scale, cache.v_scale), (*source, *first)):
            x.copy_(y)
        for (seq, rows, new), begin, stream, room in zip(parts, starts_of, side, scratch):
            stream.wait_stream(main)
            with torch.cuda.stream(stream):
                cache.append(*[x[rows] for x in given], turned[rows], cos_d, sin_d, table[seq], begin, kv[seq])
                cache.attend(turned[rows], out[rows], table[seq], begin, kv[seq], new, scratch=room)
            main.wait_stream(stream)
        cache.gather(*back, table, starts)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        calls()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        calls()
    rotated = ref.append(q, k, v, cos, sin, batch.table, batch.q_start, batch.kv_len, d, False).astype(np.float16)
    want, bound = ref.attend(rotated, batch.table, batch.q_start, batch.kv_len)
    for _ in range(5):
        compare(out, want, bound)
        same(cache, ref)
        for b in range(3):
            at = slice(int(starts[b]), int(starts[b + 1]))
            assert np.array_equal(back[0][at].cpu().numpy(), ref.values(batch.table[b], int(batch.kv_len[b]))[0].reshape(-1, kv_heads * d).astype(np.float32).astype(np.float16))
        for x in (out, turned, *back, cache.k, cache.v):
            x.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
    ops.device_status(device())
