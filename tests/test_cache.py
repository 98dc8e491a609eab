"""The 8-bit key/value cache: quantising write, read back, and streaming attention over it.

Codes and scales are compared for equality with the same formula in torch's
IEEE arithmetic; against the unrounded values in 64 bits a value read back is
off by half a step of its code (e4m3: 2^-4 of it, or 2^-10 of the scale where
the code is subnormal; int8: half the scale), 2^-22 for the 32-bit product and
division, and half a step of the 16-bit type.
"""
import pytest
import torch

DEV = "cuda"
MOST = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}


def rows(seed, *shape, dtype=torch.bfloat16, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype)


def lens(*v):
    return torch.tensor(v, dtype=torch.int32)


def quantise(x, stored):
    """(codes, scale) of rows [..., D], on the CPU."""
    most = torch.tensor(MOST[stored])
    amax = x.float().abs().amax(-1).clamp_min(2.0 ** -100)
    y = x.float() * (most / amax)[..., None]
    codes = y.round().clamp(-127, 127).to(torch.int8) if stored == torch.int8 else y.clamp(-448, 448).to(stored)
    return codes, amax * (1.0 / most)


def tables(seed, batch, per, extra=2):
    g = torch.Generator().manual_seed(seed)
    return torch.randperm(batch * per + extra, generator=g)[:batch * per].view(batch, per).to(torch.int32)


def new_cache(pages, page_rows, heads, dim, stored):
    from powershard_b200.cache import KVCache
    return KVCache(pages, page_rows, heads, dim, stored, DEV)


def bits(t):
    return t.cpu().view(torch.uint8)


# ------------------------------------------------------------------ refusals (CPU)
def test_refusals_before_any_launch():
    from powershard_b200.cache import KVCache, StreamingAttention
    from powershard_b200.contract import UnsupportedAttention
    k = torch.zeros(4, 16, 2, 128, dtype=torch.int8)
    cache = KVCache.over(k, k, torch.zeros(4, 16, 2), torch.zeros(4, 16, 2))
    with pytest.raises(ValueError):
        KVCache(0, 16, 2)
    for dim, dtype in ((96, torch.int8), (128, torch.float16), (128, torch.float8_e5m2)):
        with pytest.raises(UnsupportedAttention):
            KVCache(4, 16, 2, dim, dtype)
    with pytest.raises(ValueError):
        StreamingAttention(cache, object())(rows(0, 1, 4, 2, 128), *[rows(1, 1, 4, 2, 128)] * 2, None, lens(0))
    x = rows(0, 1, 4, 2, 128)
    for start, context in ((5, 8), (5, 12), (-1, None)):  # 5 rows held and 4 new ones are 9
        with pytest.raises(ValueError):
            StreamingAttention(cache, object())(x, x, x, None, start, context=context)
    with pytest.raises(UnsupportedAttention):  # forward only
        StreamingAttention(cache, object())(x, x.clone().requires_grad_(), x, None, 0)
    from powershard_b200 import ops
    with pytest.raises(UnsupportedAttention):  # CPU tensors
        ops.cache_write((k, k), (cache.k_scale,) * 2, (rows(0, 1, 4, 2, 128),) * 2, lens(0)[None])


def test_entries_validate_on_the_host():
    from powershard_b200 import _lib
    lib = _lib.load()
    from powershard_b200.ops import _CACHE_CALL

    def call(write=True, dtype=_lib.BF16, stored=_lib.E4M3, n=4, heads=2, dim=128, page_rows=16, pages=16, rows=16,
             strides=(0, 256, 128) * 2, table=16, count=16):
        fn = lib.ps_b200_cache_write if write else lib.ps_b200_cache_read
        return fn(_CACHE_CALL.pack(pages, 16, 16, 16, rows, 16, table, 0, count, *strides, dtype, stored, 1, n, heads,
                                   dim, 4, page_rows, 4, 4), None)

    for write in (True, False):
        assert call(write, dtype=_lib.FP32) == _lib.ERR_UNSUPPORTED
        assert call(write, stored=_lib.BF16) == _lib.ERR_UNSUPPORTED
        assert call(write, dim=96) == _lib.ERR_UNSUPPORTED and b"64, 128 or 256" in lib.ps_b200_last_error()
        assert call(write, page_rows=0) == _lib.ERR_INVALID and call(write, n=1 << 32) == _lib.ERR_INVALID and call(write, heads=5000) == _lib.ERR_INVALID
        assert call(write, pages=24) == _lib.ERR_INVALID and call(write, rows=24) == _lib.ERR_INVALID
        assert call(write, strides=(0, 250, 128) * 2) == _lib.ERR_INVALID
        assert call(write, table=0) == _lib.ERR_INVALID and call(write, table=18) == _lib.ERR_INVALID
        assert call(write, n=0) == _lib.OK
    assert call(False, strides=(0, 0, 128) * 2) == _lib.ERR_INVALID and call(False, strides=(0, 256, 0) * 2) == _lib.ERR_INVALID
    assert call(False, count=0) == _lib.ERR_INVALID and b"lengths" in lib.ps_b200_last_error()
    assert lib.ps_b200_kernel_launches() == 0


def test_streaming_refuses_a_page_table_too_short():
    from powershard_b200.cache import KVCache, StreamingAttention
    from powershard_b200.sparse import SparseProvider
    k = torch.zeros(4, 16, 2, 128, dtype=torch.int8)
    cache = KVCache.over(k, k, torch.zeros(4, 16, 2), torch.zeros(4, 16, 2))
    x = rows(0, 1, 4, 2, 128)
    for table in (torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, 0, dtype=torch.int32)):
        for start, context in ((29, None), (lens(3), 33)):
            with pytest.raises(ValueError, match="page table"):
                StreamingAttention(cache, SparseProvider(1.0))(x, x, x, table, start, context=context)


def test_cache_refuses_what_autograd_would_record():
    from powershard_b200.cache import KVCache
    from powershard_b200.contract import UnsupportedAttention
    k = torch.zeros(4, 16, 2, 128, dtype=torch.int8)
    cache = KVCache.over(k, k, torch.zeros(4, 16, 2), torch.zeros(4, 16, 2))
    x, leaf = rows(0, 1, 4, 2, 128), rows(0, 1, 4, 2, 128).requires_grad_()
    for a, b in ((leaf, x), (x, leaf)):
        with pytest.raises(UnsupportedAttention, match="grad"):
            cache.write(a, b, lens(0)[None])
        with pytest.raises(UnsupportedAttention, match="grad"):
            cache.read(lens(0)[None], lens(4), a, b)


def test_forward_mode_tangents_are_refused():
    import torch.autograd.forward_ad as fwd
    from powershard_b200 import sparse
    from powershard_b200.cache import KVCache
    from powershard_b200.contract import UnsupportedAttention
    k = torch.zeros(4, 16, 2, 128, dtype=torch.int8)
    cache = KVCache.over(k, k, torch.zeros(4, 16, 2), torch.zeros(4, 16, 2))
    x, m = rows(0, 1, 4, 2, 128), torch.zeros(1, 2, 2, 128)
    with fwd.dual_level():
        d, dm = fwd.make_dual(x, x), fwd.make_dual(m, m)
        for call in (lambda: cache.write(x, d, lens(0)[None]), lambda: cache.read(lens(0)[None], lens(4), d, x),
                     lambda: sparse._no_grad(x, d), lambda: sparse._no_grad(dm)):
            with pytest.raises(UnsupportedAttention, match="tangent"):
                call()
        sparse._no_grad(x, m)


# ------------------------------------------------------------------ write and read
@pytest.mark.gpu
@pytest.mark.parametrize("stored", [torch.float8_e4m3fn, torch.int8])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("batch,n,heads,dim,page_rows", [
    (1, 1, 1, 128, 16), (3, 1, 5, 64, 7), (2, 37, 3, 128, 16), (1, 300, 40, 128, 128), (2, 65, 12, 256, 48),
    (1, 9, 200, 64, 1)])
def test_write_then_read(cuda_lib, stored, dtype, batch, n, heads, dim, page_rows):
    per = -(-(n + 11) // page_rows)
    table = tables(1, batch, per)
    cache = new_cache(batch * per + 2, page_rows, heads, dim, stored)
    k, v = rows(2, batch, n, heads, dim, dtype=dtype), rows(3, batch, n, heads, dim, dtype=dtype, scale=30.0)
    k[0, 0, 0] = 0  # a row of zeros
    v[0, n - 1, heads - 1, 0] = 1e-7 if dtype == torch.float16 else 1e-36
    start, used = lens(*range(7, 7 + batch)), lens(*[n if b == 0 else n // 2 for b in range(batch)])
    before = bits(cache.k)
    cache.write(k.to(DEV), v.to(DEV), table.to(DEV), start.to(DEV), used.to(DEV))
    ck, cs = quantise(k, stored)
    want, scales = before.clone(), torch.zeros(cache.k_scale.shape)
    for b in range(batch):
        for i in range(int(used[b])):
            p = int(start[b]) + i
            at = int(table[b, p // page_rows]), p % page_rows
            want[at], scales[at] = ck[b, i].view(torch.uint8), cs[b, i]
    assert torch.equal(bits(cache.k), want) and torch.equal(cache.k_scale.cpu(), scales)

    held = (start + used).to(DEV)
    out = [torch.full((batch, n + 5, heads, dim), 7.0, dtype=dtype, device=DEV) for _ in range(2)]
    cache.read(table.to(DEV), held, *out, first=start.to(DEV))
    for x, y in ((k, out[0]), (v, out[1])):
        codes, scale = quantise(x, stored)
        back = (codes.float() * scale[..., None]).to(dtype)
        y = y.cpu()
        for b in range(batch):
            u = int(used[b])
            assert torch.equal(y[b, :u], back[b, :u])
            assert (y[b, u:] == 7.0).all()  # behind the sequence: as it was
            err = (y[b, :u].double() - x[b, :u].double()).abs()
            s = x[b, :u].double().abs().amax(-1, keepdim=True) / MOST[stored]
            half = 0.5 * s if stored == torch.int8 else torch.maximum(2.0 ** -4 * x[b, :u].double().abs(), 2.0 ** -10 * s)
            tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
            bound = half * (1 + 2.0 ** -20) + (2.0 ** -22 + torch.finfo(dtype).eps / 2) * 1.1 * x[b, :u].double().abs()
            bound = bound + (torch.finfo(dtype).eps / 2) * half + tiny + 2.0 ** -100
            assert (err <= bound).all()


@pytest.mark.gpu
@pytest.mark.parametrize("stored", [torch.float8_e4m3fn, torch.int8])
def test_positions_without_a_page(cuda_lib, stored):
    """Rows outside the table, before position 0 or on a page that does not exist are dropped; read back they are zeros."""
    cache = new_cache(3, 8, 2, 128, stored)
    table = torch.tensor([[0, 5, -1, 2]], dtype=torch.int32, device=DEV)
    k = rows(4, 1, 40, 2, 128).to(DEV)
    cache.write(k, k, table, lens(-3).to(DEV))
    out = [torch.full((1, 40, 2, 128), 3.0, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    cache.read(table, lens(39).to(DEV), *out)
    codes, scale = quantise(k.cpu(), stored)
    back = (codes.float() * scale[..., None]).to(torch.bfloat16)
    got = out[0].cpu()
    assert torch.equal(got[0, :8], back[0, 3:11]) and torch.equal(got[0, 24:32], back[0, 27:35])
    assert not got[0, 8:24].any() and not got[0, 32:39].any() and (got[0, 39] == 3.0).all()
    assert not bits(cache.k[1]).any()  # the page that no table names


@pytest.mark.gpu
@pytest.mark.parametrize("stored", [torch.float8_e4m3fn, torch.int8])
def test_rows_with_nan_and_inf_read_back_as_nan(cuda_lib, stored):
    cache = new_cache(1, 8, 3, 128, stored)
    k = rows(5, 1, 3, 3, 128)
    k[0, 0, 0, 3], k[0, 1, 1, 127], k[0, 2, 2, 0] = float("nan"), float("inf"), float("-inf")
    table = lens(0)[None].to(DEV)
    cache.write(k.to(DEV), k.to(DEV), table)
    out = [torch.empty(1, 3, 3, 128, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    cache.read(table, lens(3).to(DEV), *out)
    bad = torch.eye(3, dtype=torch.bool)[None, :, :, None].expand(1, 3, 3, 128)
    assert torch.equal(torch.isnan(out[0].cpu()), bad)


@pytest.mark.gpu
def test_strided_rows_and_a_shared_pool(cuda_lib):
    """Rows that are views into a fused projection; a layer's pages that are a slice of one pool; a page table
    that is a slice of a longer one; sequences that share their first pages."""
    from powershard_b200.cache import KVCache
    pool = torch.zeros(2, 2, 10, 16, 3, 128, dtype=torch.int8, device=DEV)  # layers, K/V, pages
    scale = torch.zeros(2, 2, 10, 16, 3, device=DEV)
    cache = KVCache.over(pool[1, 0], pool[1, 1], scale[1, 0], scale[1, 1])
    qkv = rows(6, 1, 40, 3, 3, 128).to(DEV)
    long = torch.full((2, 9), -1, dtype=torch.int32)
    long[0, :3], long[1, :3] = torch.tensor([4, 1, 7]), torch.tensor([4, 1, 2])
    long = long.to(DEV)
    cache.write(qkv[:, :, 1], qkv[:, :, 2], long[:1, :3])
    out = [torch.empty(2, 5, 40, 128, dtype=torch.float16, device=DEV).transpose(1, 2)[:, :, 1:4] for _ in range(2)]
    cache.read(long[:, :3], lens(40, 32).to(DEV), *out)
    codes, s = quantise(qkv[0, :, 2].cpu(), torch.int8)
    back = (codes.float() * s[..., None]).half()
    assert torch.equal(out[1][0].cpu(), back) and torch.equal(out[1][1, :32].cpu(), back[:32])
    assert not pool[0].any()


@pytest.mark.gpu
def test_strides_of_axes_of_one(cuda_lib):
    """The stride of an axis with one entry says nothing."""
    for n, heads in ((9, 2), (1, 2), (9, 1)):
        x = rows(7, 1, n, heads, 128).to(DEV)
        st = [3 if m == 1 else s for m, s in zip(x.shape, x.stride())]
        cache, table, out = new_cache(1, 16, heads, 128, torch.int8), lens(0)[None].to(DEV), [torch.zeros_like(x) for _ in range(2)]
        cache.write(x.as_strided(x.shape, st), x, table)
        cache.read(table, lens(n).to(DEV), out[0].as_strided(x.shape, st), out[1])
        assert torch.equal(*out) and out[0].any()


@pytest.mark.gpu
def test_offsets_past_32_bits(cuda_lib):
    """A pool of more than 2^32 codes: rows on its last pages."""
    pages = 2 ** 32 // (256 * 16 * 128) + 3
    cache = new_cache(pages, 256, 16, 128, torch.int8)
    assert cache.k.numel() > 2 ** 32
    k, v = rows(50, 1, 300, 16, 128), rows(51, 1, 300, 16, 128)
    table = torch.tensor([[pages - 1, pages - 2]], dtype=torch.int32, device=DEV)
    cache.write(k.to(DEV), v.to(DEV), table)
    out = [torch.empty(1, 300, 16, 128, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    cache.read(table, lens(300).to(DEV), *out)
    for x, y in ((k, out[0]), (v, out[1])):
        codes, s = quantise(x, torch.int8)
        assert torch.equal(y.cpu(), (codes.float() * s[..., None]).to(torch.bfloat16))
    assert not cache.k[:pages - 2].any()


@pytest.mark.gpu
def test_autograd_sees_what_a_call_overwrites(cuda_lib):
    """A tensor that autograd keeps for a backward pass and that read or write changes is noticed, as after any
    other operation in place; inference tensors have no such count."""
    cache = new_cache(2, 16, 2, 128, torch.int8)
    table = lens(0)[None].to(DEV)
    x = rows(90, 1, 4, 2, 128).to(DEV)
    out = [torch.zeros_like(x) for _ in range(2)]
    leaf = torch.ones((), device=DEV, dtype=x.dtype, requires_grad=True)
    for i in range(2):
        y = (leaf * out[i]).sum()
        cache.read(table, lens(4).to(DEV), *out)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()
    wide = torch.ones((), device=DEV, requires_grad=True)
    y = (wide * cache.k_scale).sum()
    cache.write(x, x, table)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    with torch.inference_mode():
        out = [torch.zeros_like(x) for _ in range(2)]
        cache.read(table, lens(4).to(DEV), *out)
    cache.read(table, lens(4).to(DEV), *out)


# ------------------------------------------------------------------ the operators together
def ref_streaming(q, k, v, keep, key_block, q_len, k_len):
    from test_sparse import ref_provider
    return ref_provider(q, k, v, keep, 256, key_block, None, q_len, k_len)


@pytest.mark.gpu
@pytest.mark.parametrize("stored", [torch.float8_e4m3fn, torch.int8])
def test_streaming_steps(cuda_lib, stored):
    """Three steps of a ragged batch: append, read back, select and attend; the keys and values attended are
    the ones the cache holds (reference on the quantised values)."""
    from powershard_b200 import sparse
    from powershard_b200.cache import StreamingAttention
    from test_sparse import assert_attention
    batch, heads, kv, page_rows, steps, n = 2, 4, 2, 48, 3, 300
    per = -(-steps * n // page_rows)
    table = tables(7, batch, per).to(DEV)
    cache = new_cache(batch * per + 2, page_rows, kv, 128, stored)
    attend = StreamingAttention(cache, sparse.SparseProvider(4, key_block=64))
    held = lens(0, 0)
    past = [[torch.empty(0, kv, 128) for _ in range(batch)] for _ in range(2)]
    for step in range(steps):
        new = lens(n, n - 150 * step)
        q, k, v = rows(10 + step, batch, n, heads, 128), rows(20 + step, batch, n, kv, 128), rows(30 + step, batch, n, kv, 128)
        got = attend(q.to(DEV), k.to(DEV), v.to(DEV), table, held.to(DEV), context=steps * n, lengths=new.to(DEV))
        for side, x in zip(past, (k, v)):
            codes, s = quantise(x, stored)
            back = (codes.float() * s[..., None]).to(torch.bfloat16)
            for b in range(batch):
                side[b] = torch.cat([side[b].to(torch.bfloat16), back[b, :int(new[b])]])
        held = held + new
        full = [torch.stack([torch.cat([x, x.new_zeros(steps * n - len(x), kv, 128)]) for x in side]) for side in past]
        want, mag = ref_streaming(q, *full, 4, 64, new, held)
        assert_attention(got, want, mag)


@pytest.mark.gpu
def test_streaming_dense_and_captured(cuda_lib):
    """A dense provider over the same cache, and a captured step replayed with new rows and lengths."""
    from powershard_b200 import sparse
    from powershard_b200.cache import StreamingAttention
    from powershard_b200.graphs import GraphedCall
    from powershard_b200.provider import B200Provider
    from test_sparse import assert_attention, ref_attention
    table = tables(8, 1, 8).to(DEV)
    cache = new_cache(10, 64, 2, 128, torch.float8_e4m3fn)
    dense = StreamingAttention(cache, B200Provider())
    with pytest.raises(ValueError):
        dense(*[rows(40, 1, 8, 2, 128).to(DEV)] * 3, table, lens(0).to(DEV), context=8)
    whole = []
    for step in range(2):
        q, k, v = (rows(41 + 3 * step + i, 1, 200, 2, 128) for i in range(3))
        out = dense(q.to(DEV), k.to(DEV), v.to(DEV), table, 200 * step)
        codes = [quantise(x, torch.float8_e4m3fn) for x in (k, v)]
        whole.append([(c.float() * s[..., None]).to(torch.bfloat16) for c, s in codes])
        ks, vs = (torch.cat([w[i] for w in whole], 1) for i in range(2))
        every = torch.arange(-(-ks.shape[1] // 128), dtype=torch.int32).expand(1, 2, 1, -1)
        assert_attention(out, *ref_attention(q, ks, vs, every))
    # the same step, captured: start and lengths are device tensors that the caller advances
    step = StreamingAttention(cache, sparse.SparseProvider(1.0, key_block=64))
    x = [t.to(DEV) for t in (q, k, v)]
    start, used = lens(200).to(DEV), lens(200).to(DEV)
    graphed = GraphedCall(step, *x, table, start, context=400, lengths=used)
    graphed()
    torch.cuda.synchronize()
    assert_attention(graphed.out, *ref_attention(q, ks, vs, every))
    q2 = rows(60, 1, 200, 2, 128)
    x[0].copy_(q2)
    start.fill_(100)
    graphed()
    torch.cuda.synchronize()
    ks2, vs2 = (torch.cat([w[0][:, :100], w[1]], 1) for w in ([a[0] for a in whole], [a[1] for a in whole]))
    every = torch.arange(3, dtype=torch.int32).expand(1, 2, 1, -1)
    assert_attention(graphed.out, *ref_attention(q2, ks2, vs2, every))


@pytest.mark.gpu
def test_streaming_lengths_beyond_the_rows(cuda_lib):
    """New rows in use are counted from 0 to the rows given: what a sequence held is neither shortened nor is
    anything attended that this step did not write (a page's earlier content)."""
    from powershard_b200 import sparse
    from powershard_b200.cache import StreamingAttention
    table = tables(9, 2, 4).to(DEV)
    q, k, v = (rows(80 + i, 2, 40, 2, 128).to(DEV) for i in range(3))
    old = [rows(83 + i, 2, 256, 2, 128, scale=5.0).to(DEV) for i in range(2)]

    def step(*used):
        cache = new_cache(10, 64, 2, 128, torch.int8)
        cache.write(*old, table)  # stale rows behind position 100, earlier tokens before it
        attend = StreamingAttention(cache, sparse.SparseProvider(1.0, key_block=64))
        return attend(q, k, v, table, lens(100, 100).to(DEV), context=256, lengths=lens(*used).to(DEV))
    assert torch.equal(step(90, -30), step(40, 0))


@pytest.mark.gpu
def test_a_refused_step_writes_nothing(cuda_lib):
    from powershard_b200 import sparse
    from powershard_b200.cache import StreamingAttention
    from powershard_b200.contract import AttentionOptions, UnsupportedAttention
    from powershard_b200.provider import B200Provider
    cache = new_cache(4, 64, 2, 128, torch.int8)
    table = lens(0, 1)[None].to(DEV)
    x = rows(91, 1, 40, 2, 128).to(DEV)
    for provider in (sparse.SparseProvider(2), B200Provider()):
        attend = StreamingAttention(cache, provider)
        for q, options in ((x, AttentionOptions(causal=True)), (x[..., :64], None), (x.float(), None), (x.cpu(), None)):
            with pytest.raises((UnsupportedAttention, ValueError)):
                attend(q, x, x, table, 0, options)
    with pytest.raises(ValueError):
        StreamingAttention(cache, sparse.SparseProvider(2))(x, x, x, table, 0, allowed=torch.ones(7, 3, dtype=torch.bool, device=DEV))
    assert not bits(cache.k).any() and not bits(cache.v).any()
