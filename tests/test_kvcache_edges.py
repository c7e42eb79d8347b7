"""More of the KV-cache operators at their edges: batches padded on the left, and what the other tests
of test_kvcache.py, whose helpers and tolerances these use, do not reach."""

import ctypes

import numpy as np
import pytest
import torch

import flash_lab
from flash_lab import _capi, ops
from test_kvcache import Cache, _host_cache, check_extend, check_rows, host64, offsets

BOTH = pytest.mark.parametrize("int8", [False, True], ids=["16bit", "int8"])
DIMS = pytest.mark.parametrize("d", [64, 128])


# ------------------------------------------------------------------------------------------------
# More rows than keys
# ------------------------------------------------------------------------------------------------

@pytest.mark.gpu
@BOTH
@DIMS
@pytest.mark.parametrize("lens", [(20, 20, 20, 64), (64, 1, 32), (33, 0, 20, 31, 200), (20, 32, 65)],
                         ids=lambda x: "-".join(map(str, x)))
def test_extend_left_padded_batches(lens, d, int8):
    # 64 rows per sequence, two tiles of 32 tokens: the first tile of up to 32 keys sees none. About
    # 768 items, five and more per CTA, short ones in runs before and after full ones.
    lens = [lens[b % len(lens)] for b in range(96)]
    check_extend(Cache(lens, 8, d, torch.bfloat16, int8, page=16), [64] * 96, 32, torch.bfloat16)


@pytest.mark.gpu
@BOTH
@DIMS
def test_extend_left_padded_batches_of_long_rows(d, int8):
    # One query head per KV head, tiles of 128 tokens: n - L from less than a tile to two tiles and more.
    rng = np.random.RandomState(7)
    lens = [int(x) for x in rng.choice([3, 100, 128, 129, 140, 255, 256, 300, 700], 60)]
    new = [int(x) for x in rng.choice([256, 250, 129, 300], 60)]
    check_extend(Cache(lens, 16, d, torch.float16, int8), new, 16, torch.float16)


@pytest.mark.gpu
@BOTH
@DIMS
def test_extend_left_padded_uniform_rows(d, int8):
    # The same as [B, n, H, D], where n is known on the host.
    lens = [(20, 20, 20, 64)[b % 4] for b in range(96)]
    cache = Cache(lens, 8, d, torch.float16, int8)
    q = torch.randn(96, 64, 32, d, device="cuda").half()
    for _ in range(3):
        out, lse = flash_lab.extend(q, cache.k, cache.v, cache.seq_lens, return_lse=True,
                                    **cache.kwargs())
        torch.cuda.synchronize()
        assert ops.device_status(0) == 0
        for b in range(96):
            k, v = cache.keys(b)
            check_rows(out[b], lse[b], q[b], k, v, True, d ** -0.5, int8)


# ------------------------------------------------------------------------------------------------
# V scales of an int8 cache
# ------------------------------------------------------------------------------------------------

def int8_cache_with_v_scales(lens, heads_kv, d, dtype, steps, zeros, **kw):
    """An int8 cache whose V rows have the scales `steps` (float64 [sum(lens)]), and codes of 0 and the
    smallest scale where `zeros`, as append_kv stores a row of zeros."""
    cache = Cache(lens, heads_kv, d, dtype, True, **kw)
    steps = np.where(zeros, 2.0 ** -100, steps).astype(np.float32)
    full = torch.from_numpy(np.repeat(steps[:, None], heads_kv, 1)).cuda()
    cache.put(cache.scales["v_scale"], full)
    gen = torch.Generator(device="cuda").manual_seed(5)
    codes = torch.randint(-127, 128, (sum(lens), heads_kv, d), device="cuda", generator=gen)
    codes[torch.from_numpy(zeros).cuda()] = 0
    cache.put(cache.v, codes.to(torch.int8))
    cache.host["v"] = codes.double().cpu().numpy() * steps.astype(np.float64)[:, None, None]
    return cache


# Where the rows of zeros lie: a third of the keys at random, the first or the last of each sequence (other
# key tiles, CTAs and warps than the rest), or all keys but one.
PLACES = {
    "mixed": lambda pos, n, rng: rng.rand(n) < 0.33,
    "first": lambda pos, n, rng: pos < n // 2,
    "last": lambda pos, n, rng: pos >= n // 2,
    "all but one": lambda pos, n, rng: pos != n // 3,
}


@pytest.mark.gpu
@DIMS
@pytest.mark.parametrize("where", PLACES)
@pytest.mark.parametrize("size", [2.0 ** 30, 2.0 ** 120, 2.0 ** -100], ids=["2^30", "2^120", "2^-100"])
@pytest.mark.parametrize("new", [1, 40, 90], ids=lambda n: f"{n}rows")
def test_extend_int8_rows_of_zeros_beside_large_ones(new, size, where, d):
    """Rows of zeros count in the row sum however large the other rows of V are. One row runs in the
    few-row kernel, 40 and 90 rows of 2 heads in items of one and of two tiles; a sequence has one to
    eight key tiles, and 60 sequences put several of them into a CTA.

    The bounds of check_rows hold. Where the terms of the sum take exponentials of their own, log2 of a
    scale r, |r| <= 127, enters an exponent and leaves it again, three roundings at magnitudes up to
    256 (2^-17 ln 2 each), and the reference point and the logarithm of the sum are two more at up to
    128 (2^-18 each), together less than 2.4e-5. Where they do not, log2 2^-100 is off by at most
    100 * 2^-22 and its exponent by two roundings (2^-18 and 2^-17), all times ln 2, and the sum by 2^-20
    of it: less than 2.6e-5.
    S is 6 and more, so (d + 8) 2^-24 S + 2^-19 alone is 2.7e-5."""
    rng = np.random.RandomState(11)
    lens = [int(x) for x in rng.randint(new + 30, 300, 60)] + [1000]
    steps = np.concatenate([size * 2.0 ** -rng.randint(0, 3, n).astype(np.float64) if size > 1 else
                            np.full(n, size) for n in lens])
    zeros = np.concatenate([PLACES[where](np.arange(n), n, rng) for n in lens])
    cache = int8_cache_with_v_scales(lens, 2, d, torch.bfloat16, steps, zeros)
    gen = torch.Generator(device="cuda").manual_seed(3)
    q = (3.0 * torch.randn(new * 61, 4, d, device="cuda", generator=gen)).bfloat16()
    for b in range(61):
        size = np.einsum("tgd,sd->tgs", np.abs(host64(q[b * new:b * new + new, :2])),
                         np.abs(cache.keys(b)[0][:31, 0])) * d ** -0.5   # keys that every row sees
        assert size.max(axis=-1).min() >= 6
    check_extend(cache, [new] * 61, 4, torch.bfloat16, q=q)


@pytest.mark.gpu
@pytest.mark.parametrize("new", [1, 40], ids=["few", "many"])
def test_extend_int8_v_scales_past_the_largest(new):
    # A V scale above 2^127, an infinite one and a NaN one make the rows that see their key NaN, in both
    # kernels; 2^127 itself is read.
    for bad in (float("inf"), float("nan"), 1.5 * 2.0 ** 127):
        cache = Cache([300], 1, 64, torch.bfloat16, True)
        cache.scales["v_scale"][0, 290] = bad
        q = torch.randn(new, 2, 64, device="cuda").bfloat16()
        out, lse = flash_lab.extend(q, cache.k, cache.v, cache.seq_lens, torch.tensor(
            [0, new], dtype=torch.int32, device="cuda"), return_lse=True, **cache.kwargs())
        first = max(0, new - 10)   # row i sees keys up to 300 - new + i
        assert torch.isnan(out[first:]).all() and torch.isnan(lse[first:]).all()
        assert torch.isfinite(out[:first]).all() and torch.isfinite(lse[:first]).all()
    zeros = np.zeros(300, dtype=bool)
    steps = np.full(300, 2.0 ** 100)
    steps[7] = 2.0 ** 127
    cache = int8_cache_with_v_scales([300], 1, 64, torch.bfloat16, steps, zeros)
    cache.v[0, 7] = (cache.v[0, 7] > 0).to(torch.int8)   # 2^127 or 0
    cache.host["v"][7] = cache.v[0, 7].double().cpu().numpy() * 2.0 ** 127
    check_extend(cache, [new], 2, torch.bfloat16)


# ------------------------------------------------------------------------------------------------
# Records of checked calls
# ------------------------------------------------------------------------------------------------

class FakeBinding:
    """The binding's records, without kernels."""

    def __init__(self):
        self.known = []

    def extend_fast(self, *args):
        return None

    def extend_known(self, *args):
        self.known.append(args)

    def decode(self, *args):
        raise AssertionError("a recorded call ran")


def test_calls_without_a_status_word_are_not_recorded(monkeypatch):
    # While a graph is captured, a device that has no status word yet gets none: a call recorded then would
    # run without one for good, and its timed-out waits would never be reported.
    q = torch.zeros(2, 4, 64, dtype=torch.float16)
    kc, vc = (torch.zeros(2, 16, 2, 64, dtype=torch.float16) for _ in range(2))
    lens = torch.full((2,), 16, dtype=torch.int32)
    status = 0
    binding = FakeBinding()
    monkeypatch.setattr(ops, "_NATIVE", binding)
    monkeypatch.setattr(ops, "DEBUG", False)
    monkeypatch.setattr(ops, "_DECODE_CALLS", {})
    monkeypatch.setattr(ops, "_status_ptr", lambda device: status)
    monkeypatch.setattr(ops, "_sm_count", lambda device: 148)
    monkeypatch.setattr(ops, "_select_cached", lambda *args: ops.DECODE_IMPLS["splitkv"])
    monkeypatch.setattr(ops, "_call_op", lambda name, q, *args: (q, q[..., 0].float()))
    monkeypatch.setattr("flash_lab.kvcache._require_kernels", lambda device: None)
    for status, records in ((0, 0), (4096, 1)):
        flash_lab.extend(q, kc, vc, lens)
        flash_lab.decode(q, kc, vc, lens)
        assert len(binding.known) == len(ops._DECODE_CALLS) == records
    assert binding.known[0][-2] == 4096 and next(iter(ops._DECODE_CALLS.values()))[3] == 4096


# ------------------------------------------------------------------------------------------------
# Offsets past the rows
# ------------------------------------------------------------------------------------------------

@pytest.mark.gpu
@BOTH
def test_append_and_extend_agree_on_offsets_past_the_rows(int8):
    # Offsets are clamped to the rows that there are: of 10 and 3 promised rows the second sequence has
    # one, and they are its last keys for append_kv as for extend.
    lens, cu = [12, 9], torch.tensor([-4, 10, 13], dtype=torch.int32, device="cuda")
    cache = Cache(lens, 2, 64, torch.float16, int8, page=8)
    k, v = (torch.randn(11, 2, 64, device="cuda").half() for _ in range(2))
    flash_lab.append_kv(k, v, cache.k, cache.v, cache.seq_lens, cu, **cache.kwargs())
    got = flash_lab.gather_kv(cache.k, cache.v, cache.seq_lens, offsets(lens), 21,
                              dtype=torch.float32 if int8 else None, **cache.kwargs())
    for x, y, name in zip(got, (k, v), "kv"):
        want = torch.from_numpy(cache.host[name]).cuda()
        want[2:12], want[20] = y[:10].double(), y[10].double()
        # int8 rows: half a step and a few fp32 roundings; values as they are otherwise.
        step = want.abs().amax(-1, keepdim=True) / 127 if int8 else 0.0
        assert ((x.double() - want).abs() <= 0.501 * step).all()
        cache.host[name] = host64(x)
    q = torch.randn(11, 4, 64, device="cuda").half()
    out, lse = flash_lab.extend(q, cache.k, cache.v, cache.seq_lens, cu, return_lse=True,
                                **cache.kwargs())
    check_rows(out[:10], lse[:10], q[:10], *cache.keys(0), True, 0.125, int8)
    check_rows(out[10:], lse[10:], q[10:], *cache.keys(1), True, 0.125, int8)


@pytest.mark.gpu
def test_append_of_fewer_rows_than_the_sequences_have():
    # rows < batch * rows_per_seq (C entry only): the last sequence has what is left, one row.
    lib = _capi.load()
    cache = Cache([6, 6], 1, 64, torch.float16, poison=False)
    before = cache.k.clone(), cache.v.clone()
    k = torch.randn(4, 1, 64, device="cuda").half()
    c = cache_struct(cache)
    r = _capi.KVRows(k.data_ptr(), k.data_ptr(), 64, 64, 64, 64, 0, cache.seq_lens.data_ptr(), 4, 3,
                     _capi.FLB_FP16)
    assert lib.flb_kv_append(ctypes.byref(c), ctypes.byref(r),
                             torch.cuda.current_stream().cuda_stream) == 0
    for x, y in zip((cache.k, cache.v), before):
        y[0, 3:6], y[1, 5] = k[:3], k[3]
        assert torch.equal(x, y)


def cache_struct(cache):
    """The C entries' view of a Cache."""
    from flash_lab import kvcache

    return kvcache._cache_struct(cache.k, cache.v, cache.seq_lens, cache.block_tables,
                                 cache.scales.get("k_scale"), cache.scales.get("v_scale"))


# ------------------------------------------------------------------------------------------------
# Nothing outside the buffers
# ------------------------------------------------------------------------------------------------

class Guarded:
    """Tensors inside larger ones whose other bytes must stay as they were."""

    def __init__(self):
        self.all = []

    def __call__(self, *shape, dtype, like=None):
        n = int(np.prod(shape))
        pad = 4096
        big = torch.full((n + 2 * pad,), 77, dtype=dtype, device="cuda")
        inside = big[pad:pad + n].view(shape)
        if like is not None:
            inside.copy_(like)
        self.all.append((big, pad, n))
        return inside

    def intact(self):
        return all((big[:pad] == 77).all() and (big[pad + n:] == 77).all()
                   for big, pad, n in self.all)


@pytest.mark.gpu
@BOTH
@pytest.mark.parametrize("cu", [[0, 64, 0, 64], [64, 0, 64, 0], [10 ** 9, -5, 10 ** 9, 3], [5, 5, 5, 5],
                                [-(2 ** 31), 2 ** 31 - 1, -1, 70], [0, 2, 4, 6]],
                         ids=lambda cu: "_".join(map(str, cu)))
def test_offsets_of_any_kind_write_only_the_outputs(cu, int8):
    """Offsets that decrease or run past the rows are no valid calls, and their rows are unspecified: the
    calls end, and nothing outside the outputs and the cache is written."""
    lib = _capi.load()
    rows, heads, heads_kv, d = 64, 8, 2, 64
    guard = Guarded()
    cache = Cache([300, 200, 100], heads_kv, d, torch.bfloat16, int8, page=16, poison=False)
    cache.k, cache.v = (guard(*x.shape, dtype=x.dtype, like=x) for x in (cache.k, cache.v))
    for name, x in cache.scales.items():
        cache.scales[name] = guard(*x.shape, dtype=torch.float32, like=x)
    kept = [x.clone() for x in (cache.k, cache.v, *cache.scales.values())]
    cu = torch.tensor(cu, dtype=torch.int32, device="cuda")
    q = torch.randn(rows, heads, d, device="cuda").bfloat16()
    o = guard(rows, heads, d, dtype=torch.bfloat16)
    lse = guard(rows, heads, dtype=torch.float32)
    need = lib.flb_extend_workspace_bytes(rows, heads, heads_kv, d, ops._sm_count(q.device))
    ws = guard(need, dtype=torch.uint8)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    stream = torch.cuda.current_stream().cuda_stream
    c = cache_struct(cache)
    p = _capi.ExtendParams(q.data_ptr(), o.data_ptr(), lse.data_ptr(), q.stride(0), q.stride(1),
                           o.stride(0), o.stride(1), cu.data_ptr(), cache.seq_lens.data_ptr(), rows, 0,
                           heads, 1, _capi.FLB_BF16, 0.125, ws.data_ptr(), need, status.data_ptr())
    assert lib.flb_extend_fwd(ctypes.byref(c), ctypes.byref(p), stream) == 0
    gathered = [guard(rows, heads_kv, d, dtype=torch.bfloat16) for _ in range(2)]
    r = _capi.KVRows(gathered[0].data_ptr(), gathered[1].data_ptr(), heads_kv * d, d, heads_kv * d, d,
                     cu.data_ptr(), cache.seq_lens.data_ptr(), rows, 0, _capi.FLB_BF16)
    assert lib.flb_kv_gather(ctypes.byref(c), ctypes.byref(r), stream) == 0
    torch.cuda.synchronize()
    assert int(status) == 0 and guard.intact()
    assert all(torch.equal(a, b) for a, b in zip(kept, (cache.k, cache.v, *cache.scales.values())))
    new = [torch.randn(rows, heads_kv, d, device="cuda").bfloat16() for _ in range(2)]
    r = _capi.KVRows(new[0].data_ptr(), new[1].data_ptr(), heads_kv * d, d, heads_kv * d, d,
                     cu.data_ptr(), cache.seq_lens.data_ptr(), rows, 0, _capi.FLB_BF16)
    assert lib.flb_kv_append(ctypes.byref(c), ctypes.byref(r), stream) == 0
    torch.cuda.synchronize()
    assert guard.intact()
    # Pages of no sequence are as they were, too.
    used = cache.block_tables[cache.block_tables < cache.outer].long().unique()
    other = torch.ones(cache.outer, dtype=torch.bool, device="cuda")
    other[used] = False
    for now, then in zip((cache.k, cache.v, *cache.scales.values()), kept):
        assert torch.equal(now[other], then[other])


# ------------------------------------------------------------------------------------------------
# Orders of strides
# ------------------------------------------------------------------------------------------------

@pytest.mark.gpu
@BOTH
@DIMS
@pytest.mark.parametrize("new", [(2, 1), (60, 40)], ids=["few", "many"])
def test_extend_of_head_major_queries(new, d, int8):
    # q as [H, T, D] seen through a transpose.
    cache = Cache([150, 90], 2, d, torch.bfloat16, int8, head_major=True)
    gen = torch.Generator(device="cuda").manual_seed(2)
    q = torch.randn(8, sum(new), d, device="cuda", generator=gen).bfloat16().transpose(0, 1)
    check_extend(cache, list(new), 8, torch.bfloat16, q=q)


@pytest.mark.gpu
@BOTH
def test_extend_of_strided_batches(int8):
    # [B, n, H, D] whose sequences lie apart, and head-major ones that cannot be flattened in place.
    cache = Cache([80, 33, 200], 2, 64, torch.float16, int8, page=8)
    gen = torch.Generator(device="cuda").manual_seed(4)
    base = torch.randn(3, 9, 4, 64, device="cuda", generator=gen).half()
    for q in (base[:, 2:7], base.transpose(1, 2).contiguous().transpose(1, 2)[:, :5]):
        for _ in range(2):   # checked, then recorded
            out, lse = flash_lab.extend(q, cache.k, cache.v, cache.seq_lens, return_lse=True,
                                        **cache.kwargs())
            assert out.shape == q.shape and lse.shape == (3, 5, 4)
            for b in range(3):
                check_rows(out[b], lse[b], q[b], *cache.keys(b), True, 0.125, int8)


@pytest.mark.gpu
@BOTH
@DIMS
@pytest.mark.parametrize("new", [1, 40], ids=["few", "many"])
def test_extend_of_expanded_tensors(new, d, int8):
    # One prefix for all sequences, one KV head for several, and queries repeated over heads or tokens:
    # the bits of the copied tensors.
    cache = Cache([200, 200, 200], 4, d, torch.bfloat16, int8, capacity=210)
    gen = torch.Generator(device="cuda").manual_seed(6)
    q = torch.randn(3 * new, 8, d, device="cuda", generator=gen).bfloat16()
    cu = offsets([new] * 3)

    def run(q, k, v, scales):
        for _ in range(2):   # checked, then recorded
            got = flash_lab.extend(q, k, v, cache.seq_lens, cu, return_lse=True, **scales)
        return got

    def same(q, views):
        copies = {name: x.contiguous() for name, x in views.items()}
        got, want = (run(x, y.pop("k"), y.pop("v"), y)
                     for x, y in ((q, dict(views)), (q.contiguous(), copies)))
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert not torch.isnan(got[0]).any()

    tensors = {"k": cache.k, "v": cache.v, **cache.scales}
    same(q, {name: x[1:2].expand_as(x) for name, x in tensors.items()})
    same(q, {name: x[:, :, 2:3].expand_as(x) for name, x in tensors.items()})
    same(q, {**tensors, "v": cache.v[:1, :, :1].expand_as(cache.v)})
    same(q[:, :1].expand_as(q), tensors)
    same(q[:1].expand_as(q), tensors)


def test_extend_refuses_overlapping_rows():
    # C entry: queries and outputs are matrices of distinct rows, keys lie apart.
    lib = _capi.load()
    good = dict(q=1 << 20, o=1 << 20, lse=1 << 20, q_row_stride=1024, q_head_stride=128,
                o_row_stride=1024, o_head_stride=128, cu_seqlens=1 << 20, seq_lens=1 << 20, rows=4,
                heads=8, dtype=_capi.FLB_BF16, softmax_scale=0.1)
    for changes in (dict(q_row_stride=0), dict(q_head_stride=0), dict(o_row_stride=0),
                    dict(o_head_stride=0)):
        p = _capi.ExtendParams(**{**good, **changes})
        assert lib.flb_extend_fwd(ctypes.byref(_host_cache()), ctypes.byref(p), None) \
            == _capi.FLB_ERR_UNSUPPORTED, changes
        assert b"stride 0" in lib.flb_last_error()
    for changes in (dict(k_seq_stride=0), dict(v_seq_stride=0)):
        p = _capi.ExtendParams(**good)
        assert lib.flb_extend_fwd(ctypes.byref(_host_cache(**changes)), ctypes.byref(p), None) \
            == _capi.FLB_ERR_UNSUPPORTED, changes
        assert b"stride 0" in lib.flb_last_error()


def test_extend_refuses_caches_expanded_along_their_keys():
    kc, vc = (torch.zeros(2, 16, 2, 64, dtype=torch.bfloat16) for _ in range(2))
    q, lens = torch.zeros(2, 4, 64, dtype=torch.bfloat16), torch.full((2,), 16, dtype=torch.int32)
    for k, v in ((kc[:, :1].expand_as(kc), vc), (kc, vc[:, :1].expand_as(vc))):
        with pytest.raises(ValueError, match="along their keys"):
            flash_lab.extend(q, k, v, lens)


# ------------------------------------------------------------------------------------------------
# In-place writes and arguments
# ------------------------------------------------------------------------------------------------

@pytest.mark.gpu
@BOTH
def test_append_raises_version_counters(int8, monkeypatch):
    # As any in-place write.
    cache = Cache([5, 9], 2, 64, torch.bfloat16, int8, poison=False)
    k = torch.randn(2, 2, 64, device="cuda").bfloat16()
    written = [cache.k, cache.v, *cache.scales.values()]
    for binding in (True, True, False):   # checked, recorded, without the binding
        if not binding:
            monkeypatch.setattr(ops, "_NATIVE", None)
        before = [x._version for x in written]
        flash_lab.append_kv(k, k, cache.k, cache.v, cache.seq_lens, **cache.kwargs())
        assert all(x._version > v for x, v in zip(written, before))
    monkeypatch.undo()
    # Tensors of inference mode have no counter.
    with torch.inference_mode():
        other = Cache([5, 9], 2, 64, torch.bfloat16, int8, poison=False)
        flash_lab.append_kv(k, k, other.k, other.v, other.seq_lens, **other.kwargs())
    flash_lab.append_kv(k, k, other.k, other.v, other.seq_lens, **other.kwargs())
    assert torch.equal(other.k, cache.k)


@pytest.mark.gpu
def test_autograd_notices_an_append():
    cache = Cache([5, 9], 2, 64, torch.float32, poison=False)
    k = torch.randn(2, 2, 64, device="cuda")
    w = torch.ones_like(cache.k, requires_grad=True)
    y = (w * cache.k).sum()   # saves the cache
    flash_lab.append_kv(k, k, cache.k, cache.v, cache.seq_lens)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_gather_total_is_an_integer():
    kc = torch.zeros(2, 16, 2, 64)
    lens, cu = torch.full((2,), 16, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    for total in (5.5, "5", None):
        with pytest.raises(TypeError, match="total must be an int"):
            flash_lab.gather_kv(kc, kc, lens, cu, total)
    for total in (np.int64(5), 5):
        with pytest.raises(ValueError, match="CUDA"):
            flash_lab.gather_kv(kc, kc, lens, cu, total)


@pytest.mark.gpu
def test_gather_compiles_without_graph_breaks():
    torch._dynamo.reset()
    cache = Cache([64, 40], 2, 64, torch.bfloat16, True, page=16, poison=False)
    cu = offsets([64, 40])

    def read(kc, vc, lens, tables, ks, vs, total):
        k, v = flash_lab.gather_kv(kc, vc, lens, cu, total, tables, ks, vs)
        return k * 2, v

    args = (cache.k, cache.v, cache.seq_lens, cache.block_tables, cache.scales["k_scale"],
            cache.scales["v_scale"])
    for total in (104, 110):
        for got, want in zip(torch.compile(read, fullgraph=True)(*args, total), read(*args, total)):
            assert torch.equal(got, want)
