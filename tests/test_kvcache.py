"""The KV-cache operators (append_kv, gather_kv, extend, decode over int8) against fp64 definitions.

Tolerances. u = eps / 2 of a type is the largest relative error of one rounding to it. extend
rounds the weights to 16 bits before the second product (u_p: q's type, fp16 over an int8 cache) and
the result once (u_o); a score is a sum of D products in fp32, off by at most (D + 8) 2^-24 times
the sum of their magnitudes, which moves a weight by twice that relatively; the exponential and
the running sums add less than 2^-19. Weights below fp16's normal range are off by at most 2^-25 of
a weight of 1, which adds at most L 2^-25 max|v|. So
    |o - ref| <= u_o (|ref| + t) + t,  t = a (u_p + 2 (D + 8) 2^-24 S + 2^-19) + L 2^-25 max|v|
with a = sum_j p_j |v_j| and S the largest sum of a row's score magnitudes (kv_oracle.extend), and
    |lse - ref| <= (D + 8) 2^-24 S + 2^-19 (1 + |ref|).
"""

import ctypes

import numpy as np
import pytest
import torch

import flash_lab
import kv_oracle
from flash_lab import _capi, ops

DTYPES = [torch.bfloat16, torch.float16]


def ids(x):
    return str(x).removeprefix("torch.").replace(" ", "")


def host64(x):
    return x.detach().double().cpu().numpy()


# ------------------------------------------------------------------------------------------------
# Caches for the GPU tests
# ------------------------------------------------------------------------------------------------

class Cache:
    """A cache of `lens` keys per sequence filled with random rows, and its sequences on the host.
    Rows that hold no key are poison: NaN (16 and 32 bits), or random codes with NaN scales."""

    def __init__(self, lens, heads_kv, d, dtype, int8=False, page=0, capacity=None, seed=0,
                 head_major=False, poison=True):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        self.lens, self.page, self.int8 = list(lens), page, int8
        cap = max([*lens, 1]) + 3 if capacity is None else capacity
        if page:
            need = [max(1, -(-n // page)) for n in lens]
            width = max(max(need), -(-cap // page))
            order = torch.randperm(sum(need) + 2, generator=torch.Generator().manual_seed(seed))
            self.block_tables = torch.full((len(lens), width), 10 ** 6, dtype=torch.int32)
            at = 0
            for b, n in enumerate(need):
                self.block_tables[b, :n] = order[at:at + n].int()
                at += n
            self.block_tables = self.block_tables.cuda()
            outer, rows = len(order), page
        else:
            self.block_tables = None
            outer, rows = len(lens), cap
        self.outer, self.rows = outer, rows
        shape = (outer, rows, heads_kv, d)

        def empty(shape, dtype, fill):
            if head_major:   # [outer, H_kv, rows, ...] storage seen through a transpose
                shape = (shape[0], shape[2], shape[1], *shape[3:])
                return torch.full(shape, fill, device="cuda", dtype=dtype).transpose(1, 2)
            return torch.full(shape, fill, device="cuda", dtype=dtype)

        nan = float("nan") if poison else 0.0
        self.seq_lens = torch.tensor(self.lens, dtype=torch.int32, device="cuda")
        self.scales = {}
        self.host = {}
        for name in "kv":
            x = torch.randn(sum(self.lens), heads_kv, d, device="cuda", generator=gen)
            x *= torch.exp2(3 * torch.rand(sum(self.lens), heads_kv, 1, device="cuda",
                                           generator=gen) - 2)
            if int8:
                cache = empty(shape, torch.int8, 77)
                scale = empty(shape[:3], torch.float32, nan)
                codes, steps = kv_oracle.quantise(host64(x))
                steps = steps.astype(np.float32)
                self.put(cache, torch.from_numpy(codes).to(torch.int8).cuda())
                self.put(scale, torch.from_numpy(steps).cuda())
                self.scales[name + "_scale"] = scale
                self.host[name] = codes * steps[..., None].astype(np.float64)
            else:
                cache = empty(shape, dtype, nan)
                x = x.to(dtype)
                self.put(cache, x)
                self.host[name] = host64(x)
            setattr(self, name, cache)

    def where(self, b, pos):
        if not self.page:
            return b, pos
        return int(self.block_tables[b, pos // self.page]), pos % self.page

    def put(self, cache, rows):
        o, r = [], []
        for b, n in enumerate(self.lens):
            for pos in range(n):
                at = self.where(b, pos) if not self.page else None
                if self.page:
                    at = (self._table[b][pos // self.page], pos % self.page)
                o.append(at[0])
                r.append(at[1])
        if o:
            cache[torch.tensor(o, device="cuda"), torch.tensor(r, device="cuda")] = rows

    @property
    def _table(self):
        if not hasattr(self, "_host_table"):
            self._host_table = self.block_tables.tolist()
        return self._host_table

    def keys(self, b):
        first = sum(self.lens[:b])
        return (self.host["k"][first:first + self.lens[b]],
                self.host["v"][first:first + self.lens[b]])

    def kwargs(self):
        return dict(block_tables=self.block_tables, **self.scales)


def offsets(counts):
    return torch.tensor([sum(counts[:i]) for i in range(len(counts) + 1)], dtype=torch.int32,
                        device="cuda")


def check_rows(out, lse, q, k, v, causal, scale, int8, lse_too=True):
    """One sequence's rows of extend against the definition (see the module's docstring)."""
    n, heads, d = q.shape
    if n == 0:
        return
    ref, ref_lse, a, size = kv_oracle.extend(host64(q), k, v, causal, scale)
    u_o = torch.finfo(q.dtype).eps / 2
    u_p = torch.finfo(torch.float16).eps / 2 if int8 else u_o
    score = (d + 8) * 2.0 ** -24 * size
    largest = np.abs(v).max(initial=0.0)
    t = a * (u_p + 2 * score[..., None] + 2.0 ** -19) + len(k) * 2.0 ** -25 * largest
    got = host64(out)
    err, allowed = np.abs(got - ref), u_o * (np.abs(ref) + t) + t
    assert np.isfinite(got).all()
    assert (err <= allowed).all(), (float((err - allowed).max()), float(err.max()))
    got_lse = host64(lse)
    hidden = np.isneginf(ref_lse)
    assert np.array_equal(np.isneginf(got_lse), hidden)
    with np.errstate(invalid="ignore"):
        off = np.abs(got_lse - ref_lse) - (score + 2.0 ** -19 * (1 + np.abs(ref_lse)))
    assert (off[~hidden] <= 0).all(), float(off[~hidden].max())


def check_extend(cache, new, heads, dtype, causal=True, scale=None, seed=1, extra_rows=0, q=None):
    d = cache.k.shape[3]
    scale = scale or d ** -0.5
    tokens = sum(new) + extra_rows
    if q is None:
        gen = torch.Generator(device="cuda").manual_seed(seed)
        q = torch.randn(tokens, heads, d, device="cuda", generator=gen).to(dtype)
    out, lse = flash_lab.extend(q, cache.k, cache.v, cache.seq_lens, offsets(new), causal=causal,
                                softmax_scale=scale, return_lse=True, **cache.kwargs())
    torch.cuda.synchronize()
    assert ops.device_status(0) == 0
    assert out.shape == q.shape and out.dtype == q.dtype
    assert lse.shape == q.shape[:2] and lse.dtype == torch.float32
    t = 0
    for b, n in enumerate(new):
        k, v = cache.keys(b)
        check_rows(out[t:t + n], lse[t:t + n], q[t:t + n], k, v, causal, scale, cache.int8)
        t += n
    # Rows behind the last sequence.
    assert (out[t:] == 0).all() and torch.isneginf(lse[t:]).all()
    return out, lse


# ------------------------------------------------------------------------------------------------
# extend
# ------------------------------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("int8", [False, True], ids=["16bit", "int8"])
@pytest.mark.parametrize("dtype", DTYPES, ids=ids)
@pytest.mark.parametrize("d", [64, 128])
def test_extend_ragged_batch(d, dtype, int8):
    # No rows, one row, more rows than keys, lengths around the tile sizes, an empty sequence.
    new = [0, 1, 5, 130, 7, 40, 300, 2]
    lens = [9, 1, 129, 130, 3, 256, 700, 0]
    check_extend(Cache(lens, 2, d, dtype, int8, page=16), new, 8, dtype, extra_rows=3)


@pytest.mark.gpu
@pytest.mark.parametrize("int8", [False, True], ids=["16bit", "int8"])
@pytest.mark.parametrize("causal", [True, False], ids=["causal", "full"])
@pytest.mark.parametrize("heads", [(1, 1), (6, 2), (5, 1), (16, 1), (12, 12), (128, 1), (71, 1)],
                         ids=ids)
def test_extend_head_layouts(heads, causal, int8):
    new, lens = [3, 37, 1], [200, 37, 450]
    check_extend(Cache(lens, heads[1], 64, torch.bfloat16, int8), new, heads[0], torch.bfloat16,
                 causal)


@pytest.mark.gpu
@pytest.mark.parametrize("int8", [False, True], ids=["16bit", "int8"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("page", [8, 16, 32, 64, 128, 192])
def test_extend_pages(page, d, int8):
    new, lens = [20, 1, 150], [333, 640, 151]
    cache = Cache(lens, 3, d, torch.float16, int8, page=page, seed=page)
    check_extend(cache, new, 6, torch.float16, causal=page != 64)


@pytest.mark.gpu
@pytest.mark.parametrize("int8", [False, True], ids=["16bit", "int8"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("new", [1, 2, 31, 64, 127, 128, 129, 255, 256, 257, 600])
def test_extend_chunk_sizes(new, d, int8):
    cache = Cache([new + 190], 1, d, torch.bfloat16, int8)
    check_extend(cache, [new], 1, torch.bfloat16)
    check_extend(cache, [new], 1, torch.bfloat16, causal=False)


@pytest.mark.gpu
@pytest.mark.parametrize("int8", [False, True], ids=["16bit", "int8"])
def test_extend_many_sequences(int8):
    # More sequences than CTAs, most of them single tokens.
    rng = np.random.RandomState(3)
    lens = [int(x) for x in rng.randint(1, 150, 400)]
    new = [1 if i % 7 else min(lens[i], 9) for i in range(400)]
    check_extend(Cache(lens, 1, 64, torch.bfloat16, int8, page=8), new, 4, torch.bfloat16)


@pytest.mark.gpu
@pytest.mark.parametrize("int8", [False, True], ids=["16bit", "int8"])
@pytest.mark.parametrize("sequences", [3, 40])
def test_extend_many_items_per_sequence(sequences, int8):
    # 64 query heads per KV head: an item is four tokens, so a sequence has dozens of them.
    new = [200 if i % 13 == 1 else i % 3 for i in range(sequences)]
    cache = Cache([n + 60 for n in new], 2, 64, torch.float16, int8)
    check_extend(cache, new, 128, torch.float16)


@pytest.mark.gpu
def test_decreasing_offsets_stay_inside_the_buffers():
    # Not a valid call: its rows are unspecified, but it ends and touches nothing else.
    cache = Cache([300, 200, 100], 2, 64, torch.bfloat16, page=16)
    q = torch.randn(64, 8, 64, device="cuda").bfloat16()
    big = torch.full((64 + 8, 8, 64), -7.0, device="cuda", dtype=torch.bfloat16)
    for cu in ([0, 64, 0, 64], [64, 0, 64, 0], [10 ** 9, -5, 10 ** 9, 3], [5, 5, 5, 5]):
        cu = torch.tensor(cu, dtype=torch.int32, device="cuda")
        out = flash_lab.extend(q, cache.k, cache.v, cache.seq_lens, cu, **cache.kwargs())
        big[4:-4] = out
        flash_lab.gather_kv(cache.k, cache.v, cache.seq_lens, cu, 70, **cache.kwargs())
        torch.cuda.synchronize()
        assert ops.device_status(0) == 0
    for b in range(3):   # the cache is as it was
        k, _ = cache.keys(b)
        got, _ = flash_lab.gather_kv(cache.k, cache.v, cache.seq_lens, offsets(cache.lens), 600,
                                     **cache.kwargs())
        first = sum(cache.lens[:b])
        assert np.array_equal(host64(got[first:first + len(k)]), k)


@pytest.mark.gpu
def test_offsets_past_32_bits():
    # Pages at the far end of pools of more than 2^31 rows' values: the same bits as in a small pool.
    page, heads_kv, d, lens = 64, 8, 128, [200, 130]
    blocks = (1 << 31) // (page * heads_kv * d) + 9
    k, v = (torch.randn(sum(lens), heads_kv, d, device="cuda").half() for _ in range(2))
    q = torch.randn(6, 16, d, device="cuda").half()
    seq_lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
    results = []
    for n in (8, blocks):
        pool = [torch.empty(n, page, heads_kv, d, dtype=torch.int8, device="cuda") for _ in range(2)]
        scales = dict(k_scale=torch.empty(n, heads_kv, page, device="cuda").transpose(1, 2),
                      v_scale=torch.empty(n, heads_kv, page, device="cuda").transpose(1, 2))
        tables = torch.tensor([[n - 1, n - 3, n - 5, n - 7], [n - 2, n - 4, n - 6, 0]],
                              dtype=torch.int32, device="cuda")
        flash_lab.append_kv(k, v, *pool, seq_lens, offsets(lens), tables, **scales)
        results.append((*flash_lab.gather_kv(*pool, seq_lens, offsets(lens), sum(lens), tables,
                                             dtype=torch.float16, **scales),
                        flash_lab.extend(q, *pool, seq_lens, offsets([5, 1]), tables, **scales),
                        flash_lab.extend(q, *pool, seq_lens, offsets([1, 5]), tables, **scales),
                        flash_lab.decode(q[:2], *pool, seq_lens, tables, **scales)))
    assert all(torch.equal(a, b) for a, b in zip(*results))


@pytest.mark.gpu
@pytest.mark.parametrize("int8", [False, True], ids=["16bit", "int8"])
def test_extend_long_context(int8):
    # One sequence's keys cut over every CTA and merged.
    cache = Cache([9001], 2, 128, torch.bfloat16, int8, page=64)
    check_extend(cache, [4], 8, torch.bfloat16)


@pytest.mark.gpu
@pytest.mark.parametrize("int8", [False, True], ids=["16bit", "int8"])
@pytest.mark.parametrize("scale", [1e-4, 3.0])
def test_extend_scales(scale, int8):
    # Weights that are nearly equal, and one key that takes all.
    cache = Cache([500], 2, 64, torch.float16, int8)
    check_extend(cache, [70], 4, torch.float16, scale=scale)


@pytest.mark.gpu
@pytest.mark.parametrize("int8", [False, True], ids=["16bit", "int8"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("new", [20, 160])
def test_extend_scores_that_grow_along_the_keys(new, d, int8):
    # The reference point of nearly every row moves at every key tile, in items of one tile (20
    # tokens) and of two, by several tiles of one CTA: 2 x 8 x about 30 of them for 148 CTAs.
    lens = [4500, 3400]
    cache = Cache(lens, 8, d, torch.bfloat16, int8)
    factor = 6.0 * (torch.arange(cache.rows, device="cuda") // 128 + 1)
    if int8:
        cache.scales["k_scale"] *= factor[None, :, None]
        steps = np.concatenate([host64(cache.scales["k_scale"][b, :n]) for b, n in enumerate(lens)])
        codes = np.concatenate([host64(cache.k[b, :n]) for b, n in enumerate(lens)])
        cache.host["k"] = codes * steps[..., None]
    else:
        cache.k *= factor[None, :, None, None].to(torch.bfloat16)
        cache.host["k"] = np.concatenate([host64(cache.k[b, :n]) for b, n in enumerate(lens)])
    check_extend(cache, [new, new], 16, torch.bfloat16)


@pytest.mark.gpu
def test_extend_int8_scales_of_any_size():
    # V rows of very different sizes, tiny and zero rows among them: the weights carry the scales.
    cache = Cache([300], 1, 64, torch.bfloat16, True)
    factor = torch.exp2(torch.arange(300, device="cuda") % 61 - 40.0)
    factor[7] = 0.0
    cache.scales["v_scale"][0, :300, 0] *= factor
    cache.host["v"] *= host64(factor)[:, None, None]
    cache.scales["v_scale"].clamp_min_(2.0 ** -100)
    check_extend(cache, [40], 2, torch.bfloat16)


@pytest.mark.gpu
@pytest.mark.parametrize("int8", [False, True], ids=["16bit", "int8"])
def test_extend_strides(int8):
    # Head-major caches (the Hugging Face layout) and q as a slice of a packed projection.
    cache = Cache([150, 90], 2, 128, torch.bfloat16, int8, head_major=True)
    packed = torch.randn(100, 12, 128, device="cuda").bfloat16()
    check_extend(cache, [60, 40], 4, torch.bfloat16, q=packed[:, 3:7])


@pytest.mark.gpu
def test_extend_uniform_rows():
    # Without offsets: the same number of rows per sequence, with the shapes of q.
    cache = Cache([80, 33, 200], 2, 64, torch.float16, page=8)
    q = torch.randn(3, 5, 4, 64, device="cuda").half()
    out, lse = flash_lab.extend(q, cache.k, cache.v, cache.seq_lens, return_lse=True,
                                **cache.kwargs())
    assert out.shape == q.shape and lse.shape == (3, 5, 4)
    flat, flat_lse = flash_lab.extend(q.flatten(0, 1), cache.k, cache.v, cache.seq_lens,
                                      offsets([5, 5, 5]), return_lse=True, **cache.kwargs())
    assert torch.equal(out.flatten(0, 1), flat) and torch.equal(lse.flatten(0, 1), flat_lse)
    one = flash_lab.extend(q[:, 4], cache.k, cache.v, cache.seq_lens, **cache.kwargs())
    assert one.shape == (3, 4, 64)
    for b in range(3):
        k, v = cache.keys(b)
        check_rows(out[b], lse[b], q[b], k, v, True, 64 ** -0.5, False)


@pytest.mark.gpu
@pytest.mark.parametrize("int8", [False, True], ids=["16bit", "int8"])
def test_extend_out_of_range_lengths_and_pages(int8):
    # Lengths are clamped to the cache; keys of pages that are no blocks of the pool are zeros
    # (of zero weight in V, a score of 0).
    lens = [40, 48]
    cache = Cache(lens, 2, 64, torch.bfloat16, int8, page=16, poison=False)
    cache.block_tables = cache.block_tables[:, :3].contiguous()
    cache.block_tables[0, 1] = -1
    for name in "kv":
        cache.host[name][16:32] = 0.0
    q = torch.randn(6, 4, 64, device="cuda").bfloat16()
    lengths = torch.tensor([40, 10 ** 9], dtype=torch.int32, device="cuda")
    out, lse = flash_lab.extend(q, cache.k, cache.v, lengths, offsets([3, 3]), return_lse=True,
                                **cache.kwargs())
    for b in range(2):
        k, v = cache.keys(b)
        check_rows(out[3 * b:3 * b + 3], lse[3 * b:3 * b + 3], q[3 * b:3 * b + 3], k, v, True, 0.125,
                   int8)
    out, lse = flash_lab.extend(q, cache.k, cache.v, torch.full_like(lengths, -5), offsets([3, 3]),
                                return_lse=True, **cache.kwargs())
    assert (out == 0).all() and torch.isneginf(lse).all()


@pytest.mark.gpu
@pytest.mark.parametrize("int8", [False, True], ids=["16bit", "int8"])
def test_extend_non_finite_values_reach_only_the_rows_that_see_them(int8):
    cache = Cache([300], 1, 64, torch.bfloat16, int8)
    q = torch.randn(40, 2, 64, device="cuda").bfloat16()
    clean = flash_lab.extend(q, cache.k, cache.v, cache.seq_lens, offsets([40]), **cache.kwargs())
    if int8:   # key 280 (row 20) unreadable in K, key 290 (row 30) in V
        cache.scales["k_scale"][0, 280] = float("nan")
        cache.scales["v_scale"][0, 290] = float("nan")
    else:
        cache.k[0, 280] = float("nan")
    out = flash_lab.extend(q, cache.k, cache.v, cache.seq_lens, offsets([40]), **cache.kwargs())
    assert torch.equal(out[:20], clean[:20])
    assert torch.isnan(out[20:]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("int8", [False, True], ids=["16bit", "int8"])
def test_extend_is_reproducible_and_ignores_its_workspace(int8):
    cache = Cache([700, 3000], 2, 128, torch.bfloat16, int8, page=32)
    q = torch.randn(90, 8, 128, device="cuda").bfloat16()
    runs = []
    for fill in (0.0, float("nan"), 1e30):
        junk = torch.full((64 << 20,), fill, device="cuda")
        torch.cuda.synchronize()
        del junk   # the allocator hands these bytes to the next call's workspace and outputs
        runs.append(flash_lab.extend(q, cache.k, cache.v, cache.seq_lens, offsets([80, 10]),
                                     return_lse=True, **cache.kwargs()))
    for out, lse in runs[1:]:
        assert torch.equal(out, runs[0][0]) and torch.equal(lse, runs[0][1])


# ------------------------------------------------------------------------------------------------
# decode over an int8 cache
# ------------------------------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("page", [0, 16, 64])
@pytest.mark.parametrize("heads", [(8, 2), (4, 4), (32, 1)], ids=ids)
@pytest.mark.parametrize("dtype", DTYPES, ids=ids)
def test_decode_int8(dtype, heads, page):
    lens = [1, 130, 2500, 64, 0, 777]
    cache = Cache(lens, heads[1], 128, dtype, True, page=page)
    q = torch.randn(6, 1, heads[0], 128, device="cuda").to(dtype)
    out, lse = flash_lab.decode(q, cache.k, cache.v, cache.seq_lens, return_lse=True,
                                **cache.kwargs())
    assert out.shape == q.shape and lse.shape == (6, heads[0])
    for b in range(6):
        k, v = cache.keys(b)
        check_rows(out[b], lse[b:b + 1], q[b], k, v, True, 128 ** -0.5, True)
    flat, flat_lse = flash_lab.decode(q[:, 0], cache.k, cache.v, cache.seq_lens, return_lse=True,
                                      **cache.kwargs())
    assert torch.equal(flat, out[:, 0]) and torch.equal(flat_lse, lse)


# ------------------------------------------------------------------------------------------------
# append_kv and gather_kv
# ------------------------------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("page", [0, 5, 16, 64])
@pytest.mark.parametrize("d,heads_kv", [(64, 1), (64, 5), (128, 3), (128, 8)])
@pytest.mark.parametrize("dtype", [*DTYPES, torch.float32], ids=ids)
def test_append_quantises_and_gather_reads_back(dtype, d, heads_kv, page):
    # A code is round(x r) with x r within 3 roundings of fp32 (2^-22 relative, at most 127) of
    # its exact value, so it is the fp64 code except at borders; the scale is two roundings off.
    new, lens = [4, 0, 1, 33, 700], [9, 3, 1, 40, 700]
    cache = Cache(lens, heads_kv, d, dtype, True, page=page, head_major=page == 16)
    tokens = sum(new)
    packed = torch.randn(tokens + 2, 3 * heads_kv, d, device="cuda").to(dtype)
    packed[1] *= 1e-3
    packed[2, :, 5] *= 100
    k, v = packed[:, heads_kv:2 * heads_kv], packed[:, 2 * heads_kv:]
    before = {name: x.clone() for name, x in
              [("k", cache.k), ("v", cache.v), *cache.scales.items()]}
    flash_lab.append_kv(k, v, cache.k, cache.v, cache.seq_lens, offsets(new), **cache.kwargs())
    written = torch.zeros(cache.outer, cache.rows, dtype=torch.bool)
    t = 0
    for b, (n, length) in enumerate(zip(new, lens)):
        for i in range(n):
            at = cache.where(b, length - n + i)
            written[at] = True
        if n:
            where = [cache.where(b, length - n + i) for i in range(n)]
            o, r = (torch.tensor(x, device="cuda") for x in zip(*where))
            for x, store, scale in ((k, cache.k, "k_scale"), (v, cache.v, "v_scale")):
                rows = host64(x[t:t + n])
                codes, steps = kv_oracle.quantise(rows)
                got, got_steps = host64(store[o, r]), host64(cache.scales[scale][o, r])
                assert (np.abs(got_steps / steps - 1) <= 2 * 2.0 ** -24 * 1.001).all()
                exact = rows / steps[..., None]
                border = np.abs(np.abs(exact - np.trunc(exact)) - 0.5) <= 127 * 2.0 ** -22
                assert ((got == codes) | (border & (np.abs(got - codes) == 1))).all()
        t += n
    # Every other row of the cache is as it was.
    keep = ~written.cuda()
    for name, x in (("k", cache.k), ("v", cache.v), *cache.scales.items()):
        now, then = x[keep], before[name][keep]
        assert torch.equal(now.nan_to_num(-1.0) if now.is_floating_point() else now,
                           then.nan_to_num(-1.0) if now.is_floating_point() else then)

    # Read back: one fp32 product and one rounding of the stored values; zeros past the lengths.
    ask = [6, 5, 1, 40, 650]
    total = sum(ask) + 2
    for out in (torch.bfloat16, torch.float16, torch.float32):
        got = flash_lab.gather_kv(cache.k, cache.v, cache.seq_lens, offsets(ask), total, dtype=out,
                                  **cache.kwargs())
        for x, store, scale in zip(got, (cache.k, cache.v), ("k_scale", "v_scale")):
            assert x.shape == (total, heads_kv, d) and x.dtype == out
            want = torch.zeros(total, heads_kv, d, device="cuda")
            t = 0
            for b, n in enumerate(ask):
                m = min(n, lens[b])
                if m:
                    where = [cache.where(b, i) for i in range(m)]
                    o, r = (torch.tensor(y, device="cuda") for y in zip(*where))
                    want[t:t + m] = store[o, r].float() * cache.scales[scale][o, r][..., None]
                t += n
            assert torch.equal(x, want.to(out))


@pytest.mark.gpu
@pytest.mark.parametrize("page", [0, 7, 32])
@pytest.mark.parametrize("dtype", [*DTYPES, torch.float32], ids=ids)
def test_append_and_gather_without_quantisation(dtype, page):
    new, lens = [3, 600, 0], [5, 602, 4]
    cache = Cache(lens, 3, 64, dtype, page=page)
    k, v = (torch.randn(603, 3, 64, device="cuda").to(dtype) for _ in range(2))
    flash_lab.append_kv(k, v, cache.k, cache.v, cache.seq_lens, offsets(new), **cache.kwargs())
    got = flash_lab.gather_kv(cache.k, cache.v, cache.seq_lens, offsets(lens), sum(lens),
                              **cache.kwargs())
    for x, y, name in zip(got, (k, v), "kv"):
        assert x.dtype == dtype
        want = torch.from_numpy(cache.host[name]).cuda().to(dtype)
        want[2:5], want[7:607] = y[:3], y[3:]
        assert torch.equal(x, want)


@pytest.mark.gpu
def test_append_special_rows():
    # Zeros, denormals, the largest finite values, infinities and NaN.
    x = torch.randn(1, 6, 1, 64, device="cuda")
    x[0, 0] = 0.0
    x[0, 1] *= 2.0 ** -126
    x[0, 2] *= torch.finfo(torch.float32).max / x[0, 2].abs().max()
    x[0, 3, 0, 9] = float("inf")
    x[0, 4, 0, 9] = float("nan")
    k_cache, v_cache = (torch.zeros(1, 6, 1, 64, dtype=torch.int8, device="cuda") for _ in range(2))
    k_scale, v_scale = (torch.zeros(1, 6, 1, device="cuda") for _ in range(2))
    lens = torch.tensor([6], dtype=torch.int32, device="cuda")
    flash_lab.append_kv(x, -x, k_cache, v_cache, lens, k_scale=k_scale, v_scale=v_scale)
    k, v = flash_lab.gather_kv(k_cache, v_cache, lens, offsets([6]), 6, k_scale=k_scale,
                               v_scale=v_scale, dtype=torch.float32)
    for got, want in ((k, x[0]), (v, -x[0])):
        assert (got[0] == 0).all()
        assert torch.isnan(got[3:5]).all()
        for i in (1, 2, 5):
            # Half a step, and six roundings (1 / a, r, x r, 1 / 127, s, q s) of at most 2^-24 of
            # the row's maximum, which is 127 steps.
            step = max(float(want[i].abs().max()) / 127, 2.0 ** -100)
            assert float((got[i].double() - want[i].double()).abs().max()) \
                <= step * (0.5 + 6 * 127 * 2.0 ** -24 * 1.001)
    assert torch.isnan(k_scale[0, 3:5]).all() and (k_cache[0, 3:5] == 0).all()
    assert float(k_scale[0, 0, 0]) == 2.0 ** -100


@pytest.mark.gpu
def test_append_skips_what_lies_outside():
    cache = Cache([16, 16], 2, 64, torch.bfloat16, page=16, poison=False)
    before = cache.k.clone(), cache.v.clone()
    k = torch.randn(2, 3, 2, 64, device="cuda").bfloat16()
    lens = torch.tensor([1, 10 ** 6], dtype=torch.int32, device="cuda")   # positions -2, -1, 0; far
    flash_lab.append_kv(k, k, cache.k, cache.v, lens, **cache.kwargs())
    at = cache.where(0, 0)
    assert torch.equal(cache.k[at], k[0, 2]) and torch.equal(cache.v[at], k[0, 2])
    cache.k[at], cache.v[at] = before[0][at], before[1][at]
    assert torch.equal(cache.k, before[0]) and torch.equal(cache.v, before[1])
    bad = torch.full_like(cache.block_tables, 10 ** 6)
    bad[1] = -3
    flash_lab.append_kv(k, k, cache.k, cache.v, cache.seq_lens, block_tables=bad)
    assert torch.equal(cache.k, before[0]) and torch.equal(cache.v, before[1])
    # Pages that are no blocks read back as zeros.
    got = flash_lab.gather_kv(cache.k, cache.v, cache.seq_lens, offsets([16, 16]), 32,
                              block_tables=bad)
    assert all((x == 0).all() for x in got)


# ------------------------------------------------------------------------------------------------
# Together
# ------------------------------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("int8", [False, True], ids=["16bit", "int8"])
def test_a_serving_loop(int8):
    """Prompts in chunks, then single tokens, through a paged cache: every step's rows against the
    definition on the values the cache holds."""
    heads, heads_kv, d, page = 8, 2, 128, 16
    chunks = [[100, 0, 37], [57, 211, 1], [1, 1, 1], [1, 1, 1]]
    lens = [sum(c[b] for c in chunks) for b in range(3)]
    width = -(-max(lens) // page)
    gen = torch.Generator(device="cuda").manual_seed(11)
    pool = (3 * width + 1, page, heads_kv, d)
    tables = torch.randperm(3 * width + 1)[:3 * width].view(3, width).int().cuda()
    kind = torch.int8 if int8 else torch.bfloat16
    k_cache, v_cache = (torch.zeros(pool, dtype=kind, device="cuda") for _ in range(2))
    scales = {}
    if int8:
        scales = {name: torch.zeros(pool[0], heads_kv, page, device="cuda").transpose(1, 2)
                  for name in ("k_scale", "v_scale")}
    done = [0, 0, 0]
    for chunk in chunks:
        done = [a + n for a, n in zip(done, chunk)]
        tokens = sum(chunk)
        q = torch.randn(tokens, heads, d, device="cuda", generator=gen).bfloat16()
        k, v = (torch.randn(tokens, heads_kv, d, device="cuda", generator=gen).bfloat16()
                for _ in range(2))
        seq_lens = torch.tensor(done, dtype=torch.int32, device="cuda")
        cu = offsets(chunk)
        flash_lab.append_kv(k, v, k_cache, v_cache, seq_lens, cu, tables, **scales)
        out, lse = flash_lab.extend(q, k_cache, v_cache, seq_lens, cu, tables, return_lse=True,
                                    **scales)
        stored = flash_lab.gather_kv(k_cache, v_cache, seq_lens, offsets(done), sum(done), tables,
                                     dtype=torch.float32 if int8 else None, **scales)
        t = first = 0
        for b, n in enumerate(chunk):
            keys, values = (host64(x[first:first + done[b]]) for x in stored)
            check_rows(out[t:t + n], lse[t:t + n], q[t:t + n], keys, values, True, d ** -0.5, int8)
            t += n
            first += done[b]
        if chunk == [1, 1, 1]:
            single = flash_lab.decode(q, k_cache, v_cache, seq_lens, tables, **scales)
            t = 2.0 * torch.finfo(torch.bfloat16).eps * float(stored[1].abs().max())
            assert float((single.float() - out.float()).abs().max()) <= t


@pytest.mark.gpu
@pytest.mark.parametrize("int8", [False, True], ids=["16bit", "int8"])
def test_append_and_extend_replay_in_a_cuda_graph(int8):
    """Two captured graphs of append + extend, replayed in turn on new data and lengths, with an
    eager call between them: the results of eager calls on the same data."""
    b, heads, heads_kv, d, cap = 3, 8, 2, 64, 900
    kind = torch.int8 if int8 else torch.float16
    kc, vc = (torch.zeros(b, cap, heads_kv, d, device="cuda").to(kind) for _ in range(2))
    scales = {}
    if int8:
        scales = {n: torch.full((b, cap, heads_kv), 0.01, device="cuda")
                  for n in ("k_scale", "v_scale")}
    q = torch.zeros(b, 2, heads, d, device="cuda", dtype=torch.float16)
    k, v = (torch.zeros(b, 2, heads_kv, d, device="cuda", dtype=torch.float16) for _ in range(2))
    lens = torch.full((b,), 700, dtype=torch.int32, device="cuda")

    def step():
        flash_lab.append_kv(k, v, kc, vc, lens, **scales)
        return flash_lab.extend(q, kc, vc, lens, return_lse=True, **scales)

    step()
    graphs = []
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for _ in range(2):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=stream):
                graphs.append((g, step()))
    torch.cuda.current_stream().wait_stream(stream)
    for i, lengths in enumerate([(700, 3, 2), (5, 900, 64), (130, 129, 128), (2, 2, 899)]):
        for x in (q, k, v):
            x.copy_(torch.randn_like(x))
        lens.copy_(torch.tensor(lengths))
        g, (out, lse) = graphs[i % 2]
        g.replay()
        want, want_lse = step()
        assert torch.equal(out, want) and torch.equal(lse, want_lse)


@pytest.mark.gpu
@pytest.mark.parametrize("int8", [False, True], ids=["16bit", "int8"])
def test_calls_on_two_streams(int8):
    cache = Cache([3000, 900], 2, 128, torch.bfloat16, int8, page=32)
    qs = [torch.randn(60, 8, 128, device="cuda").bfloat16() for _ in range(2)]
    cu = offsets([50, 10])
    want = [flash_lab.extend(q, cache.k, cache.v, cache.seq_lens, cu, **cache.kwargs()) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in qs]
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(flash_lab.extend(qs[i], cache.k, cache.v, cache.seq_lens, cu,
                                               **cache.kwargs()))
    torch.cuda.synchronize()
    assert ops.device_status(0) == 0
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])


@pytest.mark.gpu
@pytest.mark.parametrize("int8", [False, True], ids=["16bit", "int8"])
def test_ctypes_and_registered_ops_match_the_binding(int8, monkeypatch):
    cache = Cache([300, 40], 2, 64, torch.float16, int8, page=8)
    q = torch.randn(24, 4, 64, device="cuda").half()
    k, v = (torch.randn(24, 2, 64, device="cuda").half() for _ in range(2))
    cu = offsets([20, 4])

    def run():
        flash_lab.append_kv(k, v, cache.k, cache.v, cache.seq_lens, cu, **cache.kwargs())
        return (*flash_lab.extend(q, cache.k, cache.v, cache.seq_lens, cu, return_lse=True,
                                  **cache.kwargs()),
                *flash_lab.gather_kv(cache.k, cache.v, cache.seq_lens, offsets([300, 40]), 340,
                                     dtype=torch.float16, **cache.kwargs()))

    want = run()
    monkeypatch.setattr(ops, "_NATIVE", None)
    got = run()
    monkeypatch.undo()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    monkeypatch.setattr(ops, "_eager_ok", lambda args: False)   # through torch.ops
    got = run()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
def test_cache_operators_compile_without_graph_breaks():
    torch._dynamo.reset()
    cache = Cache([64, 40], 2, 64, torch.bfloat16, True, page=16, poison=False)
    q = torch.randn(2, 4, 64, device="cuda").bfloat16()
    k = torch.randn(2, 2, 64, device="cuda").bfloat16()

    def step(q, k, kc, vc, lens, tables, ks, vs):
        flash_lab.append_kv(k, k, kc, vc, lens, None, tables, ks, vs)
        return flash_lab.decode(q, kc, vc, lens, tables, k_scale=ks, v_scale=vs) * 2

    args = (q, k, cache.k, cache.v, cache.seq_lens, cache.block_tables, cache.scales["k_scale"],
            cache.scales["v_scale"])
    want = step(*args)
    torch.testing.assert_close(torch.compile(step, fullgraph=True)(*args), want)


@pytest.mark.gpu
def test_extend_writes_only_its_outputs():
    lib = _capi.load()
    cache = Cache([150, 1, 77], 2, 64, torch.bfloat16)
    new = [70, 1, 7]
    rows, heads, d = 78, 8, 64
    q = torch.randn(rows, heads, d, device="cuda").bfloat16()
    big = torch.full((rows + 4, heads + 2, d + 64), -7.0, device="cuda", dtype=torch.bfloat16)
    o = big[2:-2, 1:-1, :d]
    lse_big = torch.full((rows * heads + 128,), -7.0, device="cuda")
    need = lib.flb_extend_workspace_bytes(rows, heads, 2, d, ops._sm_count(q.device))
    ws = torch.full((need // 4 + 256,), -7.0, device="cuda")
    cu = offsets(new)
    c = _capi.KVCache(cache.k.data_ptr(), cache.v.data_ptr(), *cache.k.stride()[:3],
                      *cache.v.stride()[:3], 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 3, 2, d,
                      cache.rows, _capi.FLB_BF16)
    p = _capi.ExtendParams(q.data_ptr(), o.data_ptr(), lse_big[64:].data_ptr(), q.stride(0),
                           q.stride(1), o.stride(0), o.stride(1), cu.data_ptr(),
                           cache.seq_lens.data_ptr(), rows, 0, heads, 1, _capi.FLB_BF16, 0.125,
                           ws.data_ptr(), need, 0)
    stream = torch.cuda.current_stream().cuda_stream
    assert lib.flb_extend_fwd(ctypes.byref(c), ctypes.byref(p), stream) == 0
    torch.cuda.synchronize()
    want, want_lse = flash_lab.extend(q, cache.k, cache.v, cache.seq_lens, cu, return_lse=True)
    assert torch.equal(o, want) and torch.equal(lse_big[64:-64].view(rows, heads), want_lse)
    mask = torch.ones_like(big, dtype=torch.bool)
    mask[2:-2, 1:-1, :d] = False
    assert (big[mask] == -7.0).all()
    assert (lse_big[:64] == -7.0).all() and (lse_big[-64:] == -7.0).all()
    assert (ws[need // 4:] == -7.0).all()


# ------------------------------------------------------------------------------------------------
# Refusals and host-side checks (no GPU)
# ------------------------------------------------------------------------------------------------

def cpu_args(dtype=torch.bfloat16, kind=None, b=2, s=16, heads_kv=2, d=64):
    kc, vc = (torch.zeros(b, s, heads_kv, d, dtype=kind or dtype) for _ in range(2))
    lens = torch.full((b,), s, dtype=torch.int32)
    return kc, vc, lens


def test_extend_refusals():
    kc, vc, lens = cpu_args()
    q = torch.zeros(6, 4, 64, dtype=torch.bfloat16)
    cu = torch.tensor([0, 2, 6], dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        flash_lab.extend(q, kc, vc, lens, cu)
    with pytest.raises(TypeError, match="cu_seqlens must be int32"):
        flash_lab.extend(q, kc, vc, lens, cu.long())
    with pytest.raises(ValueError, match="cu_seqlens must have shape"):
        flash_lab.extend(q, kc, vc, lens, cu[:2])
    with pytest.raises(ValueError, match="must be \\[T, H, D\\]"):
        flash_lab.extend(q[None], kc, vc, lens, cu)
    with pytest.raises(ValueError, match="batch size mismatch"):
        flash_lab.extend(q, kc, vc, lens)
    with pytest.raises(ValueError, match="multiple of KV heads"):
        flash_lab.extend(q[:, :3], kc, vc, lens, cu)
    with pytest.raises(TypeError, match="q must be one of"):
        flash_lab.extend(q.half(), kc, vc, lens, cu)
    with pytest.raises(TypeError, match="q must be one of"):
        flash_lab.extend(q.float(), kc.float(), vc.float(), lens, cu)
    with pytest.raises(ValueError, match="head_dim mismatch"):
        flash_lab.extend(q[..., :32], kc, vc, lens, cu)
    with pytest.raises(ValueError, match="head_dim 32"):
        flash_lab.extend(q[..., :32], kc[..., :32], vc[..., :32], lens, cu)
    with pytest.raises(ValueError, match="softmax_scale"):
        flash_lab.extend(q, kc, vc, lens, cu, softmax_scale=-1.0)
    with pytest.raises(ValueError, match="softmax_scale"):
        flash_lab.extend(q, kc, vc, lens, cu, softmax_scale=float("inf"))
    with pytest.raises(ValueError, match="empty input"):
        flash_lab.extend(q[:0], kc, vc, lens, cu)
    with pytest.raises(ValueError, match="page_size 24"):
        flash_lab.extend(q, torch.zeros(9, 24, 2, 64).bfloat16(), torch.zeros(9, 24, 2, 64).bfloat16(),
                         lens, cu, torch.zeros(2, 3, dtype=torch.int32))
    with pytest.raises(ValueError, match="block_tables must be"):
        flash_lab.extend(q, kc, vc, lens, cu, torch.zeros(3, 3, dtype=torch.int32))
    with pytest.raises(ValueError, match="query heads per KV head"):
        flash_lab.extend(torch.zeros(6, 129, 64).bfloat16(), kc[:, :, :1], vc[:, :, :1], lens, cu)
    with pytest.raises(ValueError, match="last dimension"):
        flash_lab.extend(torch.zeros(6, 4, 128).bfloat16()[..., ::2], kc, vc, lens, cu)
    with pytest.raises(ValueError, match="one device"):
        flash_lab.extend(q.to("meta"), kc, vc, lens, cu)
    with pytest.raises(TypeError, match="torch.Tensor"):
        flash_lab.extend([1.0], kc, vc, lens, cu)


def test_int8_cache_refusals():
    kc, vc, lens = cpu_args(kind=torch.int8)
    q = torch.zeros(2, 4, 64, dtype=torch.bfloat16)
    scale = torch.ones(2, 16, 2)
    with pytest.raises(ValueError, match="int8 caches need"):
        flash_lab.extend(q, kc, vc, lens)
    with pytest.raises(ValueError, match="int8 caches need"):
        flash_lab.extend(q, kc, vc, lens, k_scale=scale)
    with pytest.raises(ValueError, match="int8 caches need"):
        flash_lab.extend(q, kc.bfloat16(), vc.bfloat16(), lens, k_scale=scale, v_scale=scale)
    with pytest.raises(TypeError, match="k_scale must be float32"):
        flash_lab.extend(q, kc, vc, lens, k_scale=scale.half(), v_scale=scale)
    with pytest.raises(ValueError, match="v_scale must have shape"):
        flash_lab.extend(q, kc, vc, lens, k_scale=scale, v_scale=scale[:, :8])
    with pytest.raises(TypeError, match="share a dtype"):
        flash_lab.extend(q, kc, vc.half(), lens, k_scale=scale, v_scale=scale)
    with pytest.raises(ValueError, match="one query token"):
        flash_lab.decode(torch.zeros(2, 2, 4, 64).half(), kc, vc, lens, k_scale=scale,
                         v_scale=scale)
    with pytest.raises(ValueError, match="impl or num_splits"):
        flash_lab.decode(q, kc, vc, lens, num_splits=2, k_scale=scale, v_scale=scale)
    with pytest.raises(ValueError, match="impl or num_splits"):
        flash_lab.decode(q, kc, vc, lens, impl="splitkv", k_scale=scale, v_scale=scale)
    with pytest.raises(ValueError, match="CUDA"):
        flash_lab.decode(q, kc, vc, lens, k_scale=scale, v_scale=scale)


def test_append_refuses_expanded_caches():
    # Sequences (or heads, for scales) that share memory would be written by several threads at once.
    kc, vc, lens = cpu_args()
    k = torch.zeros(2, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="k_cache is written"):
        flash_lab.append_kv(k, k, kc[:1].expand(2, -1, -1, -1), vc, lens)
    scale = torch.ones(2, 16, 2)
    with pytest.raises(ValueError, match="v_scale is written"):
        flash_lab.append_kv(k, k, kc.to(torch.int8), vc.to(torch.int8), lens, k_scale=scale,
                            v_scale=scale[..., :1].expand(-1, -1, 2))


def test_append_and_gather_refusals():
    kc, vc, lens = cpu_args()
    k = torch.zeros(2, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        flash_lab.append_kv(k, k, kc, vc, lens)
    with pytest.raises(ValueError, match="same shape"):
        flash_lab.append_kv(k, k[:1], kc, vc, lens)
    with pytest.raises(TypeError, match="share the cache's dtype"):
        flash_lab.append_kv(k.half(), k.half(), kc, vc, lens)
    with pytest.raises(ValueError, match="k and v rows are"):
        flash_lab.append_kv(k[:, :1], k[:, :1], kc, vc, lens)
    with pytest.raises(ValueError, match="same shape"):
        flash_lab.append_kv(k, k, kc, vc[:, :8], lens)
    with pytest.raises(ValueError, match="batch size mismatch"):
        flash_lab.append_kv(k[:1], k[:1], kc, vc, lens)
    with pytest.raises(ValueError, match="seq_lens must be 1-D"):
        flash_lab.append_kv(k, k, kc, vc, lens[:, None])
    cu = torch.tensor([0, 4, 8], dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        flash_lab.gather_kv(kc, vc, lens, cu, 8)
    with pytest.raises(ValueError, match="total must be positive"):
        flash_lab.gather_kv(kc, vc, lens, cu, 0)
    with pytest.raises(TypeError, match="cu_seqlens"):
        flash_lab.gather_kv(kc, vc, lens, None, 8)
    with pytest.raises(TypeError, match="dtype must be"):
        flash_lab.gather_kv(kc, vc, lens, cu, 8, dtype=torch.float32)
    with pytest.raises(ValueError, match="head_dim 32"):
        flash_lab.gather_kv(kc[..., :32], vc[..., :32], lens, cu, 8)


def test_registered_schemas_and_fake_kernels():
    from torch._subclasses.fake_tensor import FakeTensorMode

    schema = str(torch.ops.flash_lab.kv_append.default._schema)
    assert "Tensor(a!) k_cache, Tensor(b!) v_cache" in schema and schema.endswith("-> ()")
    with FakeTensorMode():
        kc = torch.empty(2, 64, 2, 128, dtype=torch.int8, device="cuda")
        s = torch.empty(2, 64, 2, device="cuda")
        lens = torch.empty(2, dtype=torch.int32, device="cuda")
        cu = torch.empty(3, dtype=torch.int32, device="cuda")
        q = torch.empty(7, 8, 128, dtype=torch.bfloat16, device="cuda")
        o, lse = torch.ops.flash_lab.extend_sm100(q, kc, kc, lens, cu, None, s, s, 0, True, 0.1)
        assert o.shape == q.shape and lse.shape == (7, 8) and lse.dtype == torch.float32
        k, v = torch.ops.flash_lab.kv_gather(kc, kc, lens, cu, None, s, s, 9, torch.float16)
        assert k.shape == v.shape == (9, 2, 128) and k.dtype == torch.float16


@pytest.mark.parametrize("struct,cls", [("flb_kv_cache", _capi.KVCache),
                                        ("flb_kv_rows", _capi.KVRows),
                                        ("flb_extend_params", _capi.ExtendParams)])
def test_struct_layout_matches_header(struct, cls, tmp_path):
    from test_capi import _c_layout

    fields = [name for name, _ in cls._fields_]
    layout = _c_layout(struct, fields, tmp_path)
    assert layout["sizeof"] == ctypes.sizeof(cls)
    assert all(layout[name] == getattr(cls, name).offset for name in fields)


def _host_cache(**changes):
    c = _capi.KVCache(1 << 20, 1 << 20, 4096, 256, 128, 4096, 256, 128)
    c.batch, c.heads_kv, c.head_dim, c.max_seqlen, c.dtype = 2, 2, 128, 16, _capi.FLB_BF16
    for name, value in changes.items():
        setattr(c, name, value)
    return c


@pytest.mark.parametrize("changes,status,message", [
    (dict(k_cache=0), _capi.FLB_ERR_INVALID_ARGUMENT, b"NULL"),
    (dict(batch=0), _capi.FLB_ERR_INVALID_ARGUMENT, b"empty cache"),
    (dict(max_seqlen=(1 << 30) + 1), _capi.FLB_ERR_UNSUPPORTED, b"S_max"),
    (dict(dtype=9), _capi.FLB_ERR_UNSUPPORTED, b"dtype code 9"),
    (dict(head_dim=96), _capi.FLB_ERR_UNSUPPORTED, b"head_dim 96"),
    (dict(dtype=_capi.FLB_INT8), _capi.FLB_ERR_INVALID_ARGUMENT, b"needs k_scale"),
    (dict(k_scale=1 << 20), _capi.FLB_ERR_INVALID_ARGUMENT, b"takes neither"),
    (dict(block_tables=1 << 20), _capi.FLB_ERR_INVALID_ARGUMENT, b"page_size 0"),
    (dict(block_tables=1 << 20, page_size=12, num_blocks=4, block_table_stride=9),
     _capi.FLB_ERR_INVALID_ARGUMENT, b"max_blocks * page_size"),
    (dict(block_tables=1 << 20, page_size=4, num_blocks=4, block_table_stride=3),
     _capi.FLB_ERR_INVALID_ARGUMENT, b"block_table_stride 3"),
    (dict(k_cache=(1 << 20) + 8), _capi.FLB_ERR_MISALIGNED, b"k_cache"),
    (dict(v_seq_stride=257), _capi.FLB_ERR_MISALIGNED, b"v_cache"),
])
def test_c_entries_refuse_bad_caches(changes, status, message):
    lib = _capi.load()
    c = _host_cache(**changes)
    rows, p = _capi.KVRows(), _capi.ExtendParams()
    for call in (lambda: lib.flb_kv_append(ctypes.byref(c), ctypes.byref(rows), None),
                 lambda: lib.flb_kv_gather(ctypes.byref(c), ctypes.byref(rows), None),
                 lambda: lib.flb_extend_fwd(ctypes.byref(c), ctypes.byref(p), None)):
        assert call() == status
        assert message in lib.flb_last_error()


def test_c_entries_refuse_bad_rows():
    lib = _capi.load()
    c = _host_cache()
    for entry in (lib.flb_kv_append, lib.flb_kv_gather):
        assert entry(None, None, None) == _capi.FLB_ERR_INVALID_ARGUMENT
        assert entry(ctypes.byref(c), None, None) == _capi.FLB_ERR_INVALID_ARGUMENT
        at = 1 << 20
        for fields, status in [((0, at, 256, 128, 256, 128, at, at, 4, 0, 0), 1),
                               ((at, at, 256, 128, 256, 128, at, at, 0, 0, 0), 1),
                               ((at, at, 256, 128, 256, 128, 0, at, 4, 0, 0), 1),
                               ((at, at, 256, 128, 256, 128, at, at, 4, 0, 3), 2),
                               ((at, at, 256, 128, 256, 128, at, at, 4, 0, 1), 2),
                               ((at, at + 2, 256, 128, 256, 128, at, at, 4, 0, 0), 3)]:
            rows = _capi.KVRows(*fields)
            assert entry(ctypes.byref(c), ctypes.byref(rows), None) == status, fields
    good = dict(q=1 << 20, o=1 << 20, lse=1 << 20, q_row_stride=1024, q_head_stride=128,
                o_row_stride=1024, o_head_stride=128, cu_seqlens=1 << 20, seq_lens=1 << 20, rows=4,
                heads=8, dtype=_capi.FLB_BF16, softmax_scale=0.1)
    for changes, status in [(dict(q=0), 1), (dict(rows=0), 1), (dict(cu_seqlens=0), 1),
                            (dict(heads=7), 1), (dict(heads=512), 2), (dict(dtype=2), 2),
                            (dict(dtype=1), 2), (dict(softmax_scale=0.0), 1),
                            (dict(softmax_scale=float("nan")), 1), (dict(q_row_stride=1023), 3),
                            (dict(o=(1 << 20) + 8), 3)]:
        p = _capi.ExtendParams(**{**good, **changes})
        assert lib.flb_extend_fwd(ctypes.byref(c), ctypes.byref(p), None) == status, changes
    paged = _host_cache(block_tables=1 << 20, page_size=4, num_blocks=4, block_table_stride=4)
    p = _capi.ExtendParams(**good)
    assert lib.flb_extend_fwd(ctypes.byref(paged), ctypes.byref(p), None) == 2
    assert b"page_size 4" in lib.flb_last_error()
