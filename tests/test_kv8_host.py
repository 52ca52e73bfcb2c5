"""What the operators over an 8-bit cache refuse before anything reaches a device. The entry points take any non-null context here: they
return before they look at it."""
import ctypes as C

import pytest

INVALID, UNSUPPORTED = -1, -4
CTX = C.c_void_p(16)   # never dereferenced by a refused call


def _cache(pkg, **changes):
    fields = dict(k=4096, v=8192 * 16, k_scale=1 << 20, v_scale=1 << 21, weight=1 << 22, slot_pos=1 << 23, batch=2, kv_heads=2, head_dim=64, capacity=128,
                  block=32, code=0)
    return pkg.Kv8Cache(**{**fields, **changes})


def _append(pkg, **changes):
    fields = dict(k=4096, v=8192, k_stride=128, v_stride=128, lengths=64, counts=64, starts=64, seen=64, refused=64, dtype=0, n=3, rows=6)
    return pkg.Kv8Append(**{**fields, **changes})


def _attend(pkg, **changes):
    fields = dict(q=4096, out=8192, q_stride=256, out_stride=256, lengths=64, counts=64, starts=64, scratch=1 << 24, scratch_bytes=1 << 30, scale=0.125,
                  dtype=0, heads=4, n=3, rows=6, max_len=100, accumulate=0)
    return pkg.Kv8Attend(**{**fields, **changes})


def _evict(pkg, **changes):
    fields = dict(lengths=64, seen=64, scratch=1 << 24, scratch_bytes=1 << 30, keep=40, sink=4, recent=8, max_len=128)
    return pkg.Kv8Evict(**{**fields, **changes})


BAD_CACHES = [dict(k=0), dict(v=0), dict(k_scale=0), dict(v_scale=0), dict(k=4097), dict(v=8), dict(k_scale=2), dict(weight=2), dict(slot_pos=1), dict(batch=0),
              dict(batch=65536), dict(kv_heads=0), dict(kv_heads=-1), dict(capacity=0), dict(capacity=120), dict(capacity=-32), dict(block=8), dict(block=48),
              dict(block=256, capacity=256), dict(code=2), dict(code=-1)]


@pytest.mark.parametrize("bad", BAD_CACHES, ids=str)
def test_caches_that_no_operator_takes(pkg, lib, bad):
    cache = _cache(pkg, **bad)
    assert lib.swlm_op_kv8_append_dev(CTX, cache, _append(pkg), None) == INVALID
    assert lib.swlm_op_kv8_attend_dev(CTX, cache, _attend(pkg), None) == INVALID
    assert lib.swlm_op_kv8_evict_dev(CTX, cache, cache, _evict(pkg), None) == INVALID
    assert b"kv8" in lib.swlm_last_error()


@pytest.mark.parametrize("dim", [0, -64, 32, 80, 96, 256])
def test_head_dimensions_without_a_kernel(pkg, lib, dim):
    cache = _cache(pkg, head_dim=dim)
    assert lib.swlm_op_kv8_append_dev(CTX, cache, _append(pkg), None) == UNSUPPORTED
    assert lib.swlm_op_kv8_attend_dev(CTX, cache, _attend(pkg), None) == UNSUPPORTED
    assert lib.swlm_op_kv8_evict_dev(CTX, cache, cache, _evict(pkg), None) == UNSUPPORTED


@pytest.mark.parametrize("bad", [dict(k=0), dict(v=0), dict(k=4104), dict(v=2), dict(k_stride=120), dict(v_stride=132), dict(k_stride=-128), dict(lengths=0),
                                 dict(lengths=66), dict(seen=0), dict(refused=65), dict(dtype=2), dict(n=0), dict(n=-3), dict(rows=-1)], ids=str)
def test_appends_that_are_refused(pkg, lib, bad):
    assert lib.swlm_op_kv8_append_dev(CTX, _cache(pkg), _append(pkg, **bad), None) == INVALID


@pytest.mark.parametrize("bad", [dict(q=0), dict(out=0), dict(q=4100), dict(out=8194), dict(q_stride=252), dict(out_stride=128), dict(lengths=0), dict(starts=63),
                                 dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(dtype=-1), dict(heads=0),
                                 dict(heads=5), dict(n=0), dict(rows=-1), dict(max_len=0), dict(accumulate=1, scratch=0), dict(accumulate=1, scratch=(1 << 24) + 8),
                                 dict(accumulate=1, scratch_bytes=16)], ids=str)
def test_attention_that_is_refused(pkg, lib, bad):
    assert lib.swlm_op_kv8_attend_dev(CTX, _cache(pkg), _attend(pkg, **bad), None) == INVALID


def test_weights_are_needed_where_they_are_added_to(pkg, lib):
    assert lib.swlm_op_kv8_attend_dev(CTX, _cache(pkg, weight=0), _attend(pkg, accumulate=1), None) == INVALID
    for missing in (dict(weight=0), dict(slot_pos=0)):
        bare = _cache(pkg, **missing)
        assert lib.swlm_op_kv8_evict_dev(CTX, bare, bare, _evict(pkg), None) == INVALID


@pytest.mark.parametrize("bad", [dict(lengths=0), dict(seen=0), dict(keep=0), dict(keep=-4), dict(sink=-1), dict(recent=-1), dict(sink=30, recent=11), dict(max_len=0),
                                 dict(scratch=0), dict(scratch=(1 << 24) + 4), dict(scratch_bytes=2 * 2 * 40 * 16 - 1)], ids=str)
def test_evictions_that_are_refused(pkg, lib, bad):
    cache = _cache(pkg)
    assert lib.swlm_op_kv8_evict_dev(CTX, cache, cache, _evict(pkg, **bad), None) == INVALID


def test_eviction_into_a_cache_that_does_not_fit(pkg, lib):
    far = dict(k=1 << 28, v=1 << 29, k_scale=1 << 30, v_scale=1 << 31, weight=1 << 32, slot_pos=1 << 33)
    for bad in (dict(batch=1), dict(kv_heads=4), dict(block=64), dict(code=1), dict(capacity=32)):
        assert lib.swlm_op_kv8_evict_dev(CTX, _cache(pkg), _cache(pkg, **{**far, **bad}), _evict(pkg), None) == INVALID
    # the same codes but other scales; codes that begin inside the first cache's
    for bad in (dict(k=4096, v=8192 * 16), dict(k=4096 + 2 * 2 * 128 * 64 - 16), dict(slot_pos=(1 << 22) + 4)):
        assert lib.swlm_op_kv8_evict_dev(CTX, _cache(pkg), _cache(pkg, **{**far, **bad}), _evict(pkg), None) == INVALID
        assert b"share" in lib.swlm_last_error()


def test_null_arguments(pkg, lib):
    cache = _cache(pkg)
    assert lib.swlm_op_kv8_append_dev(None, cache, _append(pkg), None) == INVALID
    assert lib.swlm_op_kv8_append_dev(CTX, None, _append(pkg), None) == INVALID
    assert lib.swlm_op_kv8_append_dev(CTX, cache, None, None) == INVALID
    assert lib.swlm_op_kv8_attend_dev(CTX, cache, None, None) == INVALID
    assert lib.swlm_op_kv8_evict_dev(CTX, cache, None, _evict(pkg), None) == INVALID
    assert lib.swlm_op_kv8_lengths_dev(CTX, 2, None, None, 1, 5, None, C.c_void_p(64), None) == INVALID
    assert lib.swlm_op_kv8_lengths_dev(CTX, 0, C.c_void_p(64), None, 1, 5, None, C.c_void_p(64), None) == INVALID
    assert lib.swlm_op_kv8_lengths_dev(CTX, 2, C.c_void_p(66), None, 1, 5, None, C.c_void_p(64), None) == INVALID


def test_scratch_sizes(pkg, lib):
    """Enough for what the kernels write: partial results of at most 64 runs of slots, the kept scores of up to 64 rows."""
    cache = _cache(pkg)
    assert lib.swlm_op_kv8_evict_scratch_bytes(cache, _evict(pkg)) == 2 * 2 * 40 * 16
    assert lib.swlm_op_kv8_attend_scratch_bytes(cache, _attend(pkg, heads=5)) == 0
    assert lib.swlm_op_kv8_evict_scratch_bytes(_cache(pkg, block=7), _evict(pkg)) == 0
    # Partial results: a place of 8, 16, 24 or 256 rows per tile and one per CTA (at most four on each of 148 SMs), or a tile's runs of slots
    # (no more than two CTAs per SM, plus one a tile); every row has its results, a maximum and a sum
    for heads, n, length in ((2, 1, 1), (8, 1, 4000), (16, 5, 8192), (8, 300, 2048)):
        wide = _cache(pkg, capacity=8192)
        rows = heads // 2 * n
        tile = 8 if rows <= 8 else 24 if rows <= 64 else 256
        tiles = 2 * 2 * -(-rows // min(tile, 16 if rows <= 64 else tile))
        plain, kept = (lib.swlm_op_kv8_attend_scratch_bytes(wide, _attend(pkg, heads=heads, n=n, max_len=length, accumulate=w, q_stride=heads * 64, out_stride=heads * 64))
                       for w in (0, 1))
        assert plain <= (tiles + 592) * (tile * (64 + 2) * 4 + 8) + 64
        assert plain == 0 or length > 128
        # weights: the scores of every slot, or the queries as fp16
        assert kept >= (2 * 2 * rows * length * 4 if rows <= 64 else 2 * 2 * rows * (64 * 2 + 8))


@pytest.mark.parametrize("batch,n,max_len", [(8192, 65537 * 256, 128), (65535, 1 << 22, 128), (8192, 1 << 29, 1 << 20)], ids=str)
def test_steps_of_more_ctas_than_a_grid_has(pkg, lib, batch, n, max_len):
    """An upper bound n whose blocks of rows, of all sequences and heads, are 2^31 or more. (Without scratch, so that nothing could be launched.)"""
    cache = _cache(pkg, batch=batch, kv_heads=8, capacity=1 << 20)
    step = _attend(pkg, heads=8, n=n, rows=batch, max_len=max_len, q_stride=512, out_stride=512, accumulate=1, scratch=0, scratch_bytes=0)
    assert lib.swlm_op_kv8_attend_scratch_bytes(cache, step) == 0
    assert lib.swlm_op_kv8_attend_dev(CTX, cache, step, None) == INVALID
    assert b"rows" in lib.swlm_last_error()


def test_steps_of_nearly_as_many_ctas_as_a_grid_has(pkg, lib):
    cache = _cache(pkg, batch=8192, kv_heads=8, capacity=1 << 20)
    step = _attend(pkg, heads=8, n=32767 * 256, rows=8192, max_len=128, q_stride=512, out_stride=512, accumulate=1)
    assert lib.swlm_op_kv8_attend_scratch_bytes(cache, step) > 0


def test_refused_must_be_aligned(pkg, lib):
    assert lib.swlm_op_kv8_attend_dev(CTX, _cache(pkg), _attend(pkg, refused=66), None) == INVALID
    assert b"4-byte" in lib.swlm_last_error()


def test_status_of_no_context(pkg, lib):
    assert lib.swlm_op_kv8_status(None) == INVALID
    assert lib.swlm_write_kv8_status(None, 1) == INVALID


SCRATCH = [
    # kv_heads, heads, head_dim, batch, n, max_len, CTAs of a launch with equal shares (0: none), rows of a tile, runs of slots of many rows
    (8, 32, 128, 8, 1, 8192, 3 * 148, 8, 0),     # a tile per (sequence, head), three CTAs on an SM
    (8, 32, 64, 41, 1, 8192, 4 * 148, 8, 0),     # four with heads of 64
    (8, 32, 128, 6, 5, 8192, 2 * 148, 16, 0),    # 20 rows: two tiles of 16, two CTAs on an SM
    (1, 4, 128, 3, 1, 8192, 3 * 64, 8, 0),       # as many CTAs as there are runs of 128 slots
    (8, 32, 128, 1, 1, 1000, 0, 8, 0),           # clusters, which join their results themselves
    (2, 2, 64, 600, 1, 256, 0, 8, 0),            # more sequences than shares are dealt of: a CTA has all slots
    (8, 32, 128, 1, 2048, 8192, 0, 256, 1),      # portions: as many CTAs as fill the GPU without runs
    (1, 4, 128, 1, 40, 8192, 0, 256, 64),        # one block of rows: a key tile per CTA
]


@pytest.mark.parametrize("accumulate", [0, 1])
@pytest.mark.parametrize("kv_heads,heads,dim,batch,n,max_len,ctas,tile,runs", SCRATCH, ids=str)
def test_scratch_is_what_the_kernels_write(pkg, lib, kv_heads, heads, dim, batch, n, max_len, ctas, tile, runs, accumulate):
    """Partial results have a place for every tile and one more per CTA of the shares, or one for every run of a tile's slots; a place has the tile's rows, each
    its results, a maximum and a sum. Weights need the kept scores of every slot and row, or the queries as fp16 with a factor and a shift each."""
    cache = _cache(pkg, kv_heads=kv_heads, head_dim=dim, batch=batch, capacity=8192)
    step = _attend(pkg, heads=heads, n=n, rows=batch * n, max_len=max_len, q_stride=heads * dim, out_stride=heads * dim, accumulate=accumulate)
    rows, groups = heads // kv_heads * n, batch * kv_heads
    tiles = groups * -(-rows // tile)
    need = (tiles + ctas) * tile * (dim + 2) * 4 + (batch + 1) * 4 if ctas else tiles * runs * tile * (dim + 2) * 4 if runs > 1 else 0
    if accumulate:
        pitch = 2 if rows <= 2 else -(-rows // 4) * 4
        need += groups * -(-max_len // 32) * 32 * pitch * 4 if rows <= 64 else tiles * tile * (dim * 2 + 8)
        need += tiles * tile * 8 if batch > 512 else 0   # (the rows' maxima and sums alone, for the launch that adds the weights)
    got = lib.swlm_op_kv8_attend_scratch_bytes(cache, step)
    assert need <= got <= need + 8 * 16


@pytest.mark.parametrize("how", [-1, 3])
def test_unknown_forms_of_the_probabilities(pkg, lib, how):
    step = _attend(pkg, probabilities=how, accumulate=1, scratch=0, scratch_bytes=0)
    assert lib.swlm_op_kv8_attend_dev(CTX, _cache(pkg), step, None) == INVALID
    assert b"probabilities" in lib.swlm_last_error() and lib.swlm_op_kv8_attend_scratch_bytes(_cache(pkg), step) == 0
