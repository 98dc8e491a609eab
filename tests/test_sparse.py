"""Block-sparse attention: block means, selection, attention over listed blocks.

The references are plain 64-bit computations on the CPU, one head and query
block at a time.  Tolerances:
* means: one rounding to fp32 (2^-24 of the mean) and the 32-bit sums of four
  values (3 * 2^-24 of the mean magnitude);
* selection: equal (whole numbers);
* attention: with A = sum p |v| / sum p, the probabilities' rounding to 16 bits
  (u = eps/2) gives u A, the output's u |out|; a score is a 32-bit sum of 128
  products, off by at most 128 * 2^-23 * sum |q k| * scale <= 2^-12 for rows of
  this size (sum |q k| * scale <= 16), which enters numerator and denominator:
  2^-11 A; the quarter of the exponentials that is computed on the FMA pipe is
  off by 2^-13.7 of its terms more, 2^-15.7 A on the average of a row and below
  the room that the worst case of the scores leaves.
"""
import math

import pytest
import torch

DEV = "cuda"


def rows(seed, *shape, dtype=torch.bfloat16, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype)


def ref_means(x, block, lengths=None):
    b, n, h, d = x.shape
    out = torch.zeros(b, -(-n // block), h, d, dtype=torch.float64)
    for i in range(b):
        used = n if lengths is None else min(max(int(lengths[i]), 0), n)
        for j in range(out.shape[1]):
            part = x[i, j * block:min((j + 1) * block, used)].double()
            if len(part):
                out[i, j] = part.mean(0)
    return out


def ref_select(q_means, k_means, keep, allowed=None, q_used=None, k_used=None):
    """q_used / k_used: blocks in use of each sequence."""
    b, nq, h, _ = q_means.shape
    nk, hk = k_means.shape[1:3]
    keep = min(keep, nk)
    blocks = torch.full((b, h, nq, keep), -1, dtype=torch.int32)
    counts = torch.zeros(b, h, nq, dtype=torch.int32)
    for i in range(b):
        for j in range(h):
            for t in range(nq if q_used is None else q_used[i]):
                s = k_means[i, :, j // (h // hk)].double() @ q_means[i, t, j].double()
                may = [n for n in range(nk if k_used is None else k_used[i])
                       if allowed is None or bool(allowed.broadcast_to(b, h, nq, nk)[i, j, t, n])]
                key = lambda n: (0 if math.isnan(s[n]) else 1, 0 if math.isnan(s[n]) else -float(s[n]), n)  # noqa: E731
                best = sorted(sorted(may, key=key)[:keep])
                counts[i, j, t] = len(best)
                blocks[i, j, t, :len(best)] = torch.tensor(best, dtype=torch.int32)
    return blocks, counts


def ref_attention(q, k, v, blocks, counts=None, query_block=256, key_block=128, scale=None, q_len=None, k_len=None):
    """(out, A) in 64 bits: A bounds what a relative error of the probabilities can move."""
    b, lq, h, d = q.shape
    lk, hk = k.shape[1:3]
    scale = d ** -0.5 if scale is None else scale
    out = torch.zeros(b, lq, h, d, dtype=torch.float64)
    mag = torch.zeros_like(out)
    for i in range(b):
        ql = lq if q_len is None else min(max(int(q_len[i]), 0), lq)
        kl = lk if k_len is None else min(max(int(k_len[i]), 0), lk)
        for j in range(h):
            for t in range(blocks.shape[2]):
                r = slice(t * query_block, min((t + 1) * query_block, ql))
                if r.start >= ql:
                    continue
                n = blocks.shape[3] if counts is None else min(max(int(counts[i, j, t]), 0), blocks.shape[3])
                at = [p for e in blocks[i, j, t, :n].tolist() if e >= 0
                      for p in range(e * key_block, min((e + 1) * key_block, kl))]
                if not at:
                    continue
                kk, vv = k[i, at, j // (h // hk)].double(), v[i, at, j // (h // hk)].double()
                p = torch.softmax(q[i, r, j].double() @ kk.T * scale, -1)
                out[i, r, j], mag[i, r, j] = p @ vv, p @ vv.abs()
    return out, mag


def assert_attention(got, want, mag):
    u = torch.finfo(got.dtype).eps / 2
    got = got.double().cpu()
    assert torch.isfinite(got).all()
    bound = (u + 2.0 ** -11) * mag + u * want.abs() + 1e-30
    worst = ((got - want).abs() / bound).max()
    assert worst <= 1.0, f"{float(worst):.2f} of the bound"


def cuda(*ts):
    return [t if t is None else t.to(DEV) for t in ts]


def lens(*v):
    return torch.tensor(v, dtype=torch.int32)


# ------------------------------------------------------------------ refusals (CPU)
def test_refusals_before_any_launch():
    from powershard_b200 import sparse
    from powershard_b200.contract import AttentionOptions, UnsupportedAttention
    x = rows(0, 1, 300, 2, 128)
    with pytest.raises(UnsupportedAttention):
        sparse.block_means(x, 64)  # CPU tensors
    with pytest.raises(UnsupportedAttention):
        sparse.sparse_attention(x, x, x, torch.zeros(1, 2, 2, 1, dtype=torch.int32))
    with pytest.raises(UnsupportedAttention):
        sparse.select_blocks(torch.zeros(1, 2, 2, 128), torch.zeros(1, 3, 2, 128), 1)
    for keep in (0, -1, 0.0, 1.5):
        with pytest.raises(ValueError):
            sparse.SparseProvider(keep)
    for blocks in ((128, 128), (256, 32), (300, 64), (256, 100)):
        with pytest.raises(ValueError):
            sparse.SparseProvider(4, query_block=blocks[0], key_block=blocks[1])
    p = sparse.SparseProvider(0.25)
    assert [p.blocks_kept(n) for n in (1, 3, 4, 5, 256)] == [1, 1, 1, 2, 64]
    assert sparse.SparseProvider(7).blocks_kept(5) == 5
    assert sparse.SparseProvider(0.07).blocks_kept(100) == 7 and sparse.SparseProvider(1e-12).blocks_kept(4) == 1
    for o in (AttentionOptions(causal=True), AttentionOptions(softmax_scale=-1.0), AttentionOptions()):
        with pytest.raises(UnsupportedAttention):
            p(x, x, x, o)  # the last one: CPU tensors


def test_public_names():
    import powershard_b200
    from powershard_b200 import cache, sparse
    assert powershard_b200.SparseProvider is sparse.SparseProvider
    assert powershard_b200.KVCache is cache.KVCache and powershard_b200.StreamingAttention is cache.StreamingAttention
    assert {"SparseProvider", "KVCache", "StreamingAttention"} <= set(powershard_b200.__all__)
    assert callable(sparse.SparseProvider(2)) and sparse.SparseProvider(2).identity["provider"] == sparse.NAME


def test_entries_validate_on_the_host():
    from powershard_b200 import _lib
    lib = _lib.load()
    import struct
    st = struct.pack("3q", 0, 256, 128)

    def fwd(dtype=_lib.BF16, heads=2, kv=2, dim=128, lq=300, lk=300, blocks=16, n=4, qb=256, kb=64, scale=0.1, q=16,
            ws=None):
        return lib.ps_b200_sparse_attn_fwd(q, st, 16, st, 16, st, 16, st, dtype, 1, heads, kv, dim, lq, lk, blocks,
                                           None, n, qb, kb, None, None, scale, ws, 0, None, None)

    assert fwd(dtype=_lib.FP32) == _lib.ERR_UNSUPPORTED
    assert fwd(dim=64) == _lib.ERR_UNSUPPORTED and b"head_dim" in lib.ps_b200_last_error()
    assert fwd(qb=128) == _lib.ERR_UNSUPPORTED and fwd(kb=32) == _lib.ERR_UNSUPPORTED
    assert fwd(heads=3) == _lib.ERR_INVALID and fwd(n=0) == _lib.ERR_INVALID and fwd(lk=0) == _lib.ERR_INVALID
    assert fwd(scale=0.0) == _lib.ERR_INVALID and fwd(scale=float("nan")) == _lib.ERR_INVALID
    assert fwd(q=18) == _lib.ERR_INVALID and fwd(blocks=None) == _lib.ERR_INVALID and fwd(blocks=18) == _lib.ERR_INVALID
    assert fwd(n=1 << 25) == _lib.ERR_INVALID  # names more than 2^30 rows
    assert fwd(lq=0) == _lib.OK

    from powershard_b200.ops import _SPARSE_CALL

    def whole(batch=1, heads=2, kv=2, dim=128, lq=300, lk=300, keep=2, qb=256, kb=64, scratch=256, nbytes=1 << 30,
              dtype=_lib.BF16):
        return lib.ps_b200_sparse_fwd(_SPARSE_CALL.pack(
            16, 16, 16, 16, 0, 0, 0, 0, scratch, 0, *(0, 256, 128) * 4, 0, 0, 0, 0, dtype, batch, heads, kv, dim, lq, lk,
            keep, qb, kb, nbytes, 0.1), None)

    assert whole(batch=1 << 31) == _lib.ERR_INVALID and whole(lk=0) == _lib.ERR_INVALID and whole(lq=0) == _lib.OK
    assert whole(keep=0) == _lib.ERR_INVALID and whole(keep=6) == _lib.ERR_INVALID and whole(heads=3) == _lib.ERR_INVALID
    assert whole(batch=60000, heads=60000, kv=60000) == _lib.ERR_UNSUPPORTED  # more blocks than can be counted
    assert whole(scratch=0) == _lib.ERR_INVALID and whole(nbytes=100) == _lib.ERR_INVALID and whole(scratch=272) == _lib.ERR_INVALID
    assert whole(dim=64) == _lib.ERR_UNSUPPORTED and whole(kb=32) == _lib.ERR_UNSUPPORTED
    assert whole(dtype=_lib.FP32) == _lib.ERR_UNSUPPORTED

    def select(heads=2, kv=2, dim=128, nq=2, nk=5, keep=3, means=16, lists=16, ws=16, nbytes=1 << 20):
        return lib.ps_b200_block_select(means, 16, 1, heads, kv, dim, nq, nk, keep, None, None, None, 256, None, 64,
                                        lists, 16, ws, nbytes, None)

    assert select(keep=0) == _lib.ERR_INVALID and select(keep=6) == _lib.ERR_INVALID
    assert select(heads=3) == _lib.ERR_INVALID and select(dim=64) == _lib.ERR_UNSUPPORTED
    assert select(nk=30000) == _lib.ERR_UNSUPPORTED and b"larger blocks" in lib.ps_b200_last_error()
    assert select(means=20) == _lib.ERR_INVALID and select(lists=None) == _lib.ERR_INVALID
    assert select(nq=0) == _lib.OK
    assert select(nk=300, ws=None) == _lib.ERR_INVALID and select(nk=300, nbytes=8) == _lib.ERR_INVALID
    need = lib.ps_b200_block_select_workspace_bytes
    assert need(1, 2, 2, 2, 300) >= 4 * 300 * 4 and need(1, 2, 2, 2, 5) == 0  # a few short lists need none

    def means(n=1, dtype=_lib.BF16, dim=128, block=64, length=100, x=16, stride=128):
        return lib.ps_b200_block_means(n, struct.pack("P", x), struct.pack("3q", 0, stride, 128), dtype, 1,
                                       struct.pack("i", length), struct.pack("i", 1), dim, struct.pack("i", block), None,
                                       struct.pack("P", 16), None)

    assert means(n=3) == _lib.ERR_INVALID and means(block=0) == _lib.ERR_INVALID and means(x=24) == _lib.ERR_INVALID
    assert means(dtype=_lib.FP32) == _lib.ERR_UNSUPPORTED and means(dim=64) == _lib.ERR_UNSUPPORTED
    assert means(stride=130) == _lib.ERR_INVALID and means(length=0) == _lib.OK
    assert lib.ps_b200_kernel_launches() == 0


def test_exponentials_of_the_other_pipe():
    """The pair of exponentials that the wide form computes without the special-function unit, step by step in 32
    bits with the constants of its source: relative error within 7.5e-5 (and the last product's 2^-24), 0 below
    -126.5, NaN kept."""
    import re
    import numpy as np
    from pathlib import Path
    import powershard_b200
    source = (Path(powershard_b200.__file__).parent / "csrc" / "ptx.cuh").read_text()
    body = source[source.index("void ex2_pair"):]
    body = body[:body.index("\n}")]
    floor = np.frombuffer(bytes.fromhex(re.search(r"0f([0-9A-F]{8})", body).group(1)), ">f4").astype(np.float32)[0]
    shift, back, *poly = [np.float32(x) for x in re.findall(r'"f"\((-?[0-9.]+)f\)', body)]
    assert back == -shift and len(poly) == 4

    def fma(a, b, c):  # one rounding: the product of two 32-bit numbers is exact in 64, the sum's rounding there is 2^-29 of a step
        return (a.astype(np.float64) * b + np.float64(c)).astype(np.float32)

    def pair(x):
        x = np.where(np.isnan(x), x, np.maximum(x, floor))
        t = x + shift
        f = x - (t + back)
        p = np.full_like(f, poly[0])
        for c in poly[1:]:
            p = fma(p, f, c)
        return p * (t.view(np.uint32) << np.uint32(23)).view(np.float32)

    x = np.concatenate([np.linspace(-126.0, 8.0, 2_000_001), np.arange(-126, 9) + 0.5, np.arange(-125, 9)]).astype(np.float32)
    got, want = pair(x).astype(np.float64), np.exp2(x.astype(np.float64))
    normal = want >= 2.0 ** -125  # below, the result may be subnormal
    assert (np.abs(got / want - 1)[normal] <= 7.5e-5 + 2.0 ** -24).all()
    assert (np.abs(got - want)[~normal] <= 7.5e-5 * want[~normal] + 2.0 ** -149).all()
    assert not pair(np.array([-np.inf, -1e30, -200.0, -127.0, -126.6], dtype=np.float32)).any()
    assert np.isnan(pair(np.array([np.nan], dtype=np.float32)))[0]


# ------------------------------------------------------------------ means
@pytest.mark.gpu
@pytest.mark.parametrize("n,heads,block", [(1, 1, 64), (300, 3, 64), (1000, 4, 256), (517, 5, 128), (130, 2, 7)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_block_means(cuda_lib, n, heads, block, dtype):
    from powershard_b200 import sparse
    x = rows(1, 2, n, heads, 128, dtype=dtype)
    used = lens(n, n // 3)
    x[1, n // 3:] = float("nan")
    got = sparse.block_means(x.to(DEV), block, used.to(DEV)).double().cpu()
    want, size = ref_means(x, block, used), ref_means(x.abs(), block, used)
    assert ((got - want).abs() <= 2.0 ** -24 * want.abs() + 3 * 2.0 ** -24 * size).all()
    strided = torch.cat([x, x], 2).transpose(1, 2).contiguous().transpose(1, 2)[:, :, :heads].to(DEV)
    assert torch.equal(sparse.block_means(strided, block, used.to(DEV)).double().cpu(), got)
    wide = x[:, :, :1].to(DEV).expand(-1, -1, 3, -1)  # heads that share their rows
    assert torch.equal(sparse.block_means(wide, block, used.to(DEV))[:, :, 2].double().cpu(), got[:, :, 0])


@pytest.mark.gpu
@pytest.mark.parametrize("n,block", [(4, 64), (1000, 256), (517, 64), (130, 7)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_block_means_of_any_values(cuda_lib, n, block, dtype):
    """Values of very different size, that cancel, subnormal, near the largest, infinite and NaN.  The means are
    64-bit sums: 1000 roundings of 2^-53 of the rows' magnitude and one of 2^-24 of the mean (2^-150 where it is
    subnormal)."""
    from powershard_b200 import sparse
    g = torch.Generator().manual_seed(35)
    span = (30, 24) if dtype == torch.bfloat16 else (14, 10)
    x = torch.randn(1, n, 3, 128, generator=g) * 2.0 ** torch.randint(-span[0], span[1], (1, n, 3, 128), generator=g)
    x[:, 1::2, 1] = -x[:, :n - n % 2:2, 1][:, :x[:, 1::2].shape[1]]  # pairs that cancel
    x = x.to(dtype)
    most = torch.finfo(dtype).max
    x[:, :, 2, 0] = most  # sums of it overflow 32 bits in bf16
    x[:, :, 2, 1] = torch.finfo(dtype).smallest_normal / 4
    x[:, ::3, 2, 2] = 0
    x[0, :4, 2, 3] = torch.tensor([60000.0, 0.0015, -60000.0, 0.0]).to(dtype)
    x[0, 4:, 2, 3] = 0
    got = sparse.block_means(x.to(DEV), block).double().cpu()
    want, size = ref_means(x, block), ref_means(x.abs(), block)
    assert ((got - want).abs() <= 2.0 ** -24 * want.abs() + 1000 * 2.0 ** -53 * size + 2.0 ** -150).all()
    x[0, n - 1, 0, 5], x[0, 0, 1, 6], x[0, n - 1, 1, 7] = math.inf, -math.inf, math.nan
    x[0, 0, 0, 8], x[0, min(block, n) - 1, 0, 8] = math.inf, -math.inf
    got, want = sparse.block_means(x.to(DEV), block).cpu(), ref_means(x, block).float()
    odd = ~torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(torch.isinf(got), torch.isinf(want))
    assert torch.equal(got[odd & ~torch.isnan(want)], want[odd & ~torch.isnan(want)])


@pytest.mark.gpu
@pytest.mark.parametrize("lq", [20, 200])
@pytest.mark.parametrize("lk", [3000, 30000])
def test_provider_means_do_not_depend_on_who_takes_them(cuda_lib, lq, lk):
    """Queries that cancel except for a few thousandths, which decide the selection: with key means kept and
    taken, few rows and more."""
    from powershard_b200 import sparse
    q, v = torch.zeros(1, lq, 2, 128, dtype=torch.float16), rows(36, 1, lk, 2, 128, dtype=torch.float16)
    q[:, 0, :, 0], q[:, 8, :, 0], q[:, 16, :, 0] = 60000.0, 0.0015, -60000.0
    q[:, 0, :, 1] = 0.0002
    k = torch.zeros(1, lk, 2, 128, dtype=torch.float16)
    k[:, 640:704, :, 0] = 1.0
    k[:, 1280:1344, :, 1] = 1.0
    p = sparse.SparseProvider(1, key_block=64)
    want = ref_provider(q, k, v, 1, 256, 64)
    args = cuda(q, k, v)
    assert_attention(p(*args), *want)
    assert_attention(p(*args, key_means=sparse.block_means(args[1], 64)), *want)


# ------------------------------------------------------------------ selection
@pytest.mark.gpu
@pytest.mark.parametrize("b,nq,nk,heads,kv,keep", [
    (1, 1, 1, 1, 1, 1), (2, 3, 7, 4, 2, 3), (1, 9, 300, 2, 2, 40), (1, 1, 513, 5, 1, 100), (2, 1, 64, 2, 2, 64),
    (1, 2, 2600, 1, 1, 260), (1, 5, 4000, 1, 1, 17), (1, 17, 33, 3, 3, 32),
    (1, 2, 256, 2, 1, 100), (2, 1, 255, 1, 1, 254), (1, 4, 97, 4, 2, 50), (1, 150, 200, 4, 2, 20)])
def test_select_blocks(cuda_lib, b, nq, nk, heads, kv, keep):
    from powershard_b200 import sparse
    qm, km = rows(2, b, nq, heads, 128, dtype=torch.float32), rows(3, b, nk, kv, 128, dtype=torch.float32)
    got = [t.cpu() for t in sparse.select_blocks(*cuda(qm, km), keep)]
    want = ref_select(qm, km, keep)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    allowed = torch.rand(nq, nk, generator=torch.Generator().manual_seed(4)) < 0.5
    allowed[0] = False  # a block of queries that may see nothing
    ql, kl = [0 if i else nq for i in range(b)], [max(1, nk - 5 * i - 1) for i in range(b)]
    got = [t.cpu() for t in sparse.select_blocks(
        *cuda(qm, km), keep, allowed=allowed.to(DEV), query_lengths=(lens(*ql) * 256).to(DEV),
        key_lengths=(lens(*kl) * 128 - 127).to(DEV))]
    want = ref_select(qm, km, keep, allowed, ql, kl)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert not got[1][:, :, 0].any() and (got[0][:, :, 0] == -1).all()


@pytest.mark.gpu
@pytest.mark.parametrize("nq", [1, 6])
@pytest.mark.parametrize("nk", [40, 400])  # the two forms of the selection
def test_select_ties_and_nan(cuda_lib, nq, nk):
    """Equal scores go to the lower index (0 and -0 among them), NaN is chosen, infinities rank as they are."""
    from powershard_b200 import sparse
    qm, km = torch.zeros(1, nq, 1, 128), torch.zeros(1, nk, 1, 128)
    qm[..., 0] = 1.0
    km[0, :, 0, 0] = torch.tensor(([0.0, -0.0] * 10 + [1.0] * 12 + [-1.0] * 8) * (nk // 40))
    for keep in (1, 5, 12, 13, 20, 32, 35, 40, nk // 2 + 1, nk):
        got = [t.cpu() for t in sparse.select_blocks(*cuda(qm, km), keep)]
        want = ref_select(qm, km, keep)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), keep
    qm[..., 1] = 1.0
    km[0, 37, 0, 0], km[0, 38, 0, 0] = float("nan"), float("-inf")
    km[0, 36, 0, 0] = float("inf")
    km[0, nk - 1, 0, 1] = float("nan")
    for keep in (1, 2, 3, 39, 40, nk - 1, nk):
        got = [t.cpu() for t in sparse.select_blocks(*cuda(qm, km), keep)]
        want = ref_select(qm, km, keep)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), keep


@pytest.mark.gpu
@pytest.mark.parametrize("nk", [40, 700, 6000])
def test_select_in_64_bits(cuda_lib, nk):
    """Scores that 32 bits cannot tell apart, few and many, and scores that overflow 32 bits."""
    from powershard_b200 import sparse
    g = torch.Generator().manual_seed(30)
    for alike in (5, 33, nk):
        qm, km = torch.randn(1, 5, 1, 128, generator=g), torch.randn(1, nk, 1, 128, generator=g)
        some = torch.randperm(nk, generator=g)[:alike]
        near = km[0, 0, 0].expand(len(some), -1).clone()
        near[torch.arange(len(some)), torch.randint(0, 128, (len(some),), generator=g)] *= 1 + 2.0 ** -22
        km[0, some, 0] = near
        order = ref_select(qm, km, nk)  # every rank at which the near ones may be cut
        for keep in (1, nk // 7, nk // 2, nk - 3):
            got = [t.cpu() for t in sparse.select_blocks(*cuda(qm, km), keep)]
            want = ref_select(qm, km, keep)
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), (alike, keep)
        for t in range(5):  # cut inside the near ones
            s = (km[0, :, 0].double() @ qm[0, t, 0].double()).sort(descending=True).values
            mid = float(km[0, some[0], 0].double() @ qm[0, t, 0].double())
            keep = min(nk, max(1, int((s > mid).sum()) + 1))
            got = sparse.select_blocks(*cuda(qm, km), keep)[0].cpu()
            assert torch.equal(got, ref_select(qm, km, keep)[0])
        assert order[1].eq(nk).all()
    for size in (1e25, 2e18, 6e17, 1e-25, 1e-38):
        qm, km = torch.randn(1, 2, 1, 128, generator=g) * size, torch.randn(1, nk, 1, 128, generator=g) * size
        got = sparse.select_blocks(*cuda(qm, km), nk // 3)[0].cpu()
        assert torch.equal(got, ref_select(qm, km, nk // 3)[0])


@pytest.mark.gpu
@pytest.mark.parametrize("q_size,k_size", [(1.0, 1e-24), (1e-24, 1.0), (1e-30, 1e10), (3e-16, 1.0), (1e-17, 1e-17)])
def test_select_of_tiny_rows(cuda_lib, q_size, k_size):
    """Rows whose squares underflow 32 bits, with neighbouring scores 2^-21 apart: nearer than 32 bits tell them."""
    from powershard_b200 import sparse
    g = torch.Generator().manual_seed(33)
    nk = 700
    step = 1 + torch.randperm(nk, generator=g).double() * 2.0 ** -21
    km = (torch.randn(1, 1, 1, 128, generator=g).double() * step[None, :, None, None] * k_size).float()
    qm = torch.randn(1, 5, 1, 128, generator=g) * q_size
    for keep in (1, 175, 400):
        got = [t.cpu() for t in sparse.select_blocks(*cuda(qm, km), keep)]
        want = ref_select(qm, km, keep)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), keep


@pytest.mark.gpu
def test_select_where_two_terms_leave_most(cuda_lib):
    """Means around 1 + 2^-8, where a second 8-bit term leaves the most (2^-17) and the product of the second
    terms is largest (2^-16), in both signs: blocks of either kind take turns in the exact order."""
    from powershard_b200 import sparse
    g = torch.Generator().manual_seed(34)
    nk = 600
    kind = torch.arange(nk) % 2  # second term just below 2^-8 and cut off, just above -2^-8 and rounded up
    base = torch.where(kind == 0, 1 + 2.0 ** -8 - 2.0 ** -16 + 2.0 ** -17 - 2.0 ** -20,
                       1 + 2.0 ** -8 + 2.0 ** -16 - 2.0 ** -17 + 2.0 ** -20).double()
    km = base[:, None].repeat(1, 128)
    flip = torch.rand(nk, 128, generator=g) < 0.02
    km = torch.where(flip, km * (1 + 2.0 ** -22), km) * (1 - 2.0 ** -21 * torch.randperm(nk, generator=g)[:, None].double())
    km = km.float()[None, :, None]
    for q in (1 + 2.0 ** -8 - 2.0 ** -17, 1 + 2.0 ** -8 + 2.0 ** -17):
        qm = torch.full((1, 3, 1, 128), q)
        qm[0, 1, :, ::2] *= -1
        for keep in (1, 150, 300, 450):
            got = sparse.select_blocks(*cuda(qm, km), keep)[0].cpu()
            assert torch.equal(got, ref_select(qm, km, keep)[0]), keep


@pytest.mark.gpu
def test_forward_only(cuda_lib):
    """What autograd would have to differentiate is refused, and runs where it records nothing."""
    from powershard_b200 import sparse
    from powershard_b200.contract import UnsupportedAttention
    x = rows(31, 1, 300, 2, 128).to(DEV)
    leaf = x.clone().requires_grad_()
    m = sparse.block_means(x, 256)
    mk = sparse.block_means(x, 128)
    lists = sparse.select_blocks(m, mk, 2)
    for call in (lambda t: sparse.block_means(t, 64), lambda t: sparse.sparse_attention(x, t, x, *lists),
                 lambda t: sparse.SparseProvider(2)(t, x, x)):
        with pytest.raises(UnsupportedAttention):
            call(leaf)
        with torch.no_grad():
            assert torch.equal(call(leaf), call(x))
    with pytest.raises(UnsupportedAttention):
        sparse.select_blocks(m.clone().requires_grad_(), mk, 2)
    for size in (0, -256):
        with pytest.raises(ValueError):
            sparse.sparse_attention(x, x, x, *lists, query_block=size)


# ------------------------------------------------------------------ attention over lists
def random_lists(seed, b, h, nq, nk, n):
    g = torch.Generator().manual_seed(seed)
    return torch.stack([torch.randperm(nk, generator=g)[:n] for _ in range(b * h * nq)]).view(b, h, nq, n).to(torch.int32)


@pytest.mark.gpu
@pytest.mark.parametrize("lq,lk,heads,kv,key_block,n", [
    (256, 256, 1, 1, 128, 1), (256, 512, 2, 2, 64, 3), (300, 1000, 2, 1, 128, 5), (1, 1, 1, 1, 64, 1),
    (1, 700, 4, 2, 64, 9), (513, 257, 2, 2, 64, 5), (130, 2000, 3, 1, 192, 10), (257, 1300, 2, 2, 256, 4),
    (70, 5000, 2, 2, 64, 70), (16, 3000, 4, 1, 128, 20), (17, 3000, 4, 1, 128, 20), (3, 640, 90, 45, 64, 5)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_sparse_attention(cuda_lib, lq, lk, heads, kv, key_block, n, dtype):
    from powershard_b200 import sparse
    b = 2
    q, k, v = (rows(s, b, m, h, 128, dtype=dtype) for s, m, h in ((5, lq, heads), (6, lk, kv), (7, lk, kv)))
    blocks = random_lists(8, b, heads, -(-lq // 256), -(-lk // key_block), n)
    got = sparse.sparse_attention(*cuda(q, k, v, blocks), key_block=key_block)
    torch.cuda.synchronize()
    sparse._status_for(got.device).check()
    assert_attention(got, *ref_attention(q, k, v, blocks, key_block=key_block))


@pytest.mark.gpu
@pytest.mark.parametrize("key_block", [64, 128])
def test_sparse_attention_lists_of_any_kind(cuda_lib, key_block):
    """Short and empty lists, entries that name no block, repeated and unordered entries, and what lies behind
    the lengths (NaN and infinities), in the whole and in the split form."""
    from powershard_b200 import sparse
    for b, heads, lq, lk, n in ((2, 3, 600, 1111, 7), (3, 2, 40, 3000, 20), (2, 3, 16, 3000, 20), (3, 60, 2, 900, 6)):
        q, k, v = (rows(s, b, m, heads, 128) for s, m in ((9, lq), (10, lk), (11, lk)))
        nq, nk = -(-lq // 256), -(-lk // key_block)
        blocks = random_lists(12, b, heads, nq, nk, n)
        blocks[0, 0, 0, :3] = torch.tensor([-1, nk, 2 ** 31 - 1])
        blocks[0, 1, 0, :] = -5                       # nothing but entries without a block
        blocks[1, 0, 0, :4] = torch.tensor([3, 3, 0, 3])  # counts each time
        blocks[1, 1, 0, 0] = nk - 1                   # the block that ends inside the tensor
        counts = torch.full((b, heads, nq), n, dtype=torch.int32)
        counts[0, 0, -1], counts[1, 1, -1], counts[1, 0, 0] = 1, 0, n + 9  # clamped to the list
        q_len, k_len = lens(lq, max(lq - 7, 1), 0)[:b], lens(lk - 70, lk, 33)[:b]
        for i in range(b):
            q[i, int(q_len[i]):] = float("nan")
            k[i, int(k_len[i]):] = float("inf")
            v[i, int(k_len[i]):] = float("nan")
        got = sparse.sparse_attention(*cuda(q, k, v, blocks, counts), key_block=key_block,
                                      query_lengths=q_len.to(DEV), key_lengths=k_len.to(DEV))
        assert_attention(got, *ref_attention(q, k, v, blocks, counts, 256, key_block, None, q_len, k_len))
        assert not got[0, :256, 1].any()  # only invalid entries: zeros
        for i in range(b):
            assert not got[i, int(q_len[i]):].any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("key_block", [64, 128])
@pytest.mark.parametrize("b,heads,lq", [(2, 70, 600), (1, 210, 257), (2, 200, 5)])
def test_units_handed_over(cuda_lib, b, heads, lq, key_block, dtype):
    """More than 400 units on at most 160 SMs, so that CTAs take unit after unit: units of two query tiles, of one
    and (few queries) of a few rows, each behind each, with lists of none, one and several key tiles."""
    from powershard_b200 import sparse
    lk, n = 700, 5
    q, k, v = (rows(s, b, m, h, 128, dtype=dtype) for s, m, h in ((70, lq, heads), (71, lk, heads // 10), (72, lk, heads // 10)))
    nq, nk = -(-lq // 256), -(-lk // key_block)
    assert b * heads * nq >= 400
    blocks = random_lists(73, b, heads, nq, nk, n)
    counts = torch.randint(0, n + 1, (b, heads, nq), generator=torch.Generator().manual_seed(74), dtype=torch.int32)
    q_len, k_len = lens(lq, lq - lq // 3)[:b], lens(lk, lk - 130)[:b]
    got = sparse.sparse_attention(*cuda(q, k, v, blocks, counts), key_block=key_block, query_lengths=q_len.to(DEV),
                                  key_lengths=k_len.to(DEV))
    torch.cuda.synchronize()
    sparse._status_for(got.device).check()
    assert_attention(got, *ref_attention(q, k, v, blocks, counts, 256, key_block, None, q_len, k_len))


@pytest.mark.gpu
def test_sparse_attention_all_blocks_is_dense(cuda_lib):
    """With every block listed in order the result is the dense kernel's."""
    from powershard_b200 import sparse
    from powershard_b200.provider import B200Provider
    q, k, v = (rows(s, 1, 1500, 4, 128).to(DEV) for s in (13, 14, 15))
    blocks = torch.arange(12, dtype=torch.int32, device=DEV).expand(1, 4, 6, 12).contiguous()
    out = sparse.sparse_attention(q, k, v, blocks, softmax_scale=0.05)
    from powershard_b200 import ops
    dense = torch.empty_like(q)
    ops.attention_blhd(q, k, v, dense, 0.05, None, None)
    # both walk the keys in the same order; only the split of the last wave differs
    err = (out.double() - dense.double()).abs().max()
    assert err <= 2 * 2.0 ** -8 * v.abs().max().double()
    assert_attention(out, *ref_attention(q.cpu(), k.cpu(), v.cpu(), blocks.cpu(), scale=0.05))
    assert isinstance(B200Provider().identity, dict)


@pytest.mark.gpu
def test_arguments_are_checked(cuda_lib):
    from powershard_b200 import sparse
    qm, km = torch.zeros(1, 2, 2, 128, device=DEV), torch.zeros(1, 3, 2, 128, device=DEV)
    with pytest.raises(ValueError):
        sparse.select_blocks(qm, km, 0)
    for bad in (dict(allowed=torch.ones(5, 3, dtype=torch.bool, device=DEV)), dict(allowed=torch.ones(2, 3, device=DEV)),
                dict(key_lengths=lens(3)), dict(key_lengths=torch.tensor([3], device=DEV)),
                dict(query_lengths=lens(3, 3).to(DEV))):
        with pytest.raises((ValueError, RuntimeError)):
            sparse.select_blocks(qm, km, 1, **bad)
    x = rows(0, 1, 300, 2, 128).to(DEV)
    ok = torch.zeros(1, 2, 2, 1, dtype=torch.int32, device=DEV)
    for q, k, lists in ((x, x[:, :, :, :64], ok), (x, x, ok.long()), (x, x, ok[:, :1]), (x, x.half(), ok), (x, x[:, :0], ok)):
        with pytest.raises((ValueError, RuntimeError)):
            sparse.sparse_attention(q, k, k, lists)
    with pytest.raises(ValueError):
        sparse.SparseProvider(1)(x, x, x, key_means=torch.zeros(1, 2, 2, 128, device=DEV))  # of another length
    assert sparse.SparseProvider(1)(x[:, :0], x, x).shape == (1, 0, 2, 128)
    from powershard_b200.contract import UnsupportedAttention
    grad = x.clone().requires_grad_()
    with pytest.raises(UnsupportedAttention):
        sparse.SparseProvider(1)(x, grad, x)
    with pytest.raises(UnsupportedAttention):
        sparse.sparse_attention(grad, x, x, ok)
    with torch.no_grad():
        assert torch.equal(sparse.SparseProvider(1)(x, grad, x), sparse.SparseProvider(1)(x, x, x))


@pytest.mark.gpu
def test_nan_keys_are_not_hidden(cuda_lib):
    from powershard_b200 import sparse
    q, k, v = (rows(s, 1, 512, 1, 128) for s in (16, 17, 18))
    for key in (0, 129, 200, 300, 3, 260, 388, 453):  # every position of a group of eight
        bad = k.clone()
        bad[0, key, 0, 5] = float("nan")
        out = sparse.SparseProvider(1)(*cuda(q, bad, v))
        assert torch.isnan(out).all(), key


@pytest.mark.gpu
@pytest.mark.parametrize("lq", [3, 300])
def test_scores_far_apart(cuda_lib, lq):
    """Scores of hundreds, most of them far below the largest: exponentials from 1 down to nothing.  A score's
    error grows with it, so the rows are chosen with products that 32 bits hold exactly."""
    from powershard_b200 import sparse
    g = torch.Generator().manual_seed(60)
    q, k = (torch.randint(-2, 3, (1, n, 2, 128), generator=g).to(torch.bfloat16) for n in (lq, 700))
    v = rows(61, 1, 700, 2, 128)
    blocks = torch.tensor([0, 3, 5, 7, 10], dtype=torch.int32).expand(1, 2, -(-lq // 256), 5).contiguous()
    for scale in (0.5, 8.0, 64.0):
        got = sparse.sparse_attention(*cuda(q, k, v, blocks), key_block=64, softmax_scale=scale)
        assert_attention(got, *ref_attention(q, k, v, blocks, key_block=64, scale=scale))


@pytest.mark.gpu
@pytest.mark.parametrize("lq", [3, 300])
def test_values_of_keys_far_away(cuda_lib, lq):
    """Keys whose probability is nothing (e^-500 and less) may hold values near the largest."""
    from powershard_b200 import sparse
    q, k = (torch.ones(1, n, 2, 128, dtype=torch.bfloat16) for n in (lq, 256))
    v = rows(63, 1, 256, 2, 128)
    far = torch.arange(256) % 3 > 0
    k[:, far] = -1.0
    v[:, far] = 1e38
    blocks = torch.tensor([0, 1], dtype=torch.int32).expand(1, 2, -(-lq // 256), 2).contiguous()
    got = sparse.sparse_attention(*cuda(q, k, v, blocks), softmax_scale=2.0)
    want, _ = ref_attention(q, k, v, blocks, scale=2.0)
    near, mag = ref_attention(q, k, torch.where(far[None, :, None, None], torch.zeros_like(v), v), blocks, scale=2.0)
    assert (want - near).abs().max() <= 1e-100
    assert_attention(got, near, mag)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,q_size,k_size", [(torch.float16, 2048.0, 3968.0), (torch.bfloat16, 8192.0, 7936.0),
                                                 (torch.float16, 2048.0, -3968.0), (torch.bfloat16, 8192.0, -7936.0)])
@pytest.mark.parametrize("b,lq,heads", [(1, 3, 2), (1, 300, 2), (2, 3, 90), (1, 300, 100)])
def test_scores_at_the_end_of_the_range(cuda_lib, b, lq, heads, dtype, q_size, k_size):
    """Scaled scores just below 2^27 (fp16) and 2^30 (bf16), all alike but for one key far behind (all products
    and sums are exact): every other key counts as much, in whichever part of a list it is."""
    from powershard_b200 import sparse
    q, k = (torch.full((b, n, h, 128), x, dtype=dtype) for n, h, x in ((lq, heads, q_size), (2000, 2, k_size)))
    k[:, 300] *= 0.75 if k_size > 0 else 1.25
    v = rows(67, b, 2000, 2, 128, dtype=dtype)
    blocks = random_lists(68, b, heads, -(-lq // 256), 31, 23)
    got = sparse.sparse_attention(*cuda(q, k, v, blocks), key_block=64)
    assert_attention(got, *ref_attention(q, k, v, blocks, key_block=64))


# ------------------------------------------------------------------ the provider
def ref_provider(q, k, v, keep, query_block=256, key_block=128, allowed=None, q_len=None, k_len=None, scale=None):
    used = lambda n, block: None if n is None else [-(-int(x) // block) for x in n]  # noqa: E731
    qm = ref_means(q, query_block, q_len).float()
    km = ref_means(k, key_block, k_len).float()
    blocks, counts = ref_select(qm, km, keep, allowed, used(q_len, query_block), used(k_len, key_block))
    return ref_attention(q, k, v, blocks, counts, query_block, key_block, scale, q_len, k_len)


@pytest.mark.gpu
@pytest.mark.parametrize("b,lq,lk,heads,kv,qb,kb,keep,ragged", [
    (1, 1000, 1000, 2, 2, 256, 128, 3, False), (2, 777, 777, 4, 2, 256, 64, 5, True), (1, 1, 4096, 3, 1, 256, 128, 8, False),
    (3, 900, 1500, 2, 1, 512, 192, 2, True), (1, 2049, 300, 1, 1, 256, 64, 5, False), (2, 7, 9000, 6, 3, 256, 64, 50, True), (4, 16, 2000, 50, 10, 256, 128, 9, True), (5, 1, 1, 2, 2, 256, 64, 1, True), (1, 200, 3000, 2, 1, 256, 128, 6, False), (2, 8, 5000, 3, 3, 256, 64, 30, False), (1, 30, 20000, 2, 1, 256, 64, 40, False),
    (2, 31, 20000, 2, 1, 256, 64, 40, True)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_provider(cuda_lib, b, lq, lk, heads, kv, qb, kb, keep, ragged, dtype):
    from powershard_b200 import sparse
    from powershard_b200.contract import AttentionOptions
    q, k, v = (rows(s, b, m, h, 128, dtype=dtype) for s, m, h in ((19, lq, heads), (20, lk, kv), (21, lk, kv)))
    k += rows(22, b, -(-lk // 64), kv, 128, dtype=dtype).repeat_interleave(64, 1)[:, :lk]
    q_len = k_len = None
    if ragged:
        q_len = lens(*[max(0, lq - i * (lq // 2 + 1)) for i in range(b)])
        k_len = lens(*[max(0, lk - i * (lk // 2 + 1)) for i in range(b)])
    p = sparse.SparseProvider(keep, query_block=qb, key_block=kb)
    got = p(*cuda(q, k, v), AttentionOptions(softmax_scale=0.07), query_lengths=None if q_len is None else q_len.to(DEV),
            key_lengths=None if k_len is None else k_len.to(DEV))
    assert got.shape == q.shape and got.dtype == dtype
    assert_attention(got, *ref_provider(q, k, v, keep, qb, kb, None, q_len, k_len, 0.07))
    if not ragged:  # kept means give the same
        kept = sparse.block_means(k.to(DEV), kb)
        again = p(*cuda(q, k, v), AttentionOptions(softmax_scale=0.07), key_means=kept)
        assert torch.equal(got, again)


@pytest.mark.gpu
def test_provider_on_strided_inputs_streams_and_graphs(cuda_lib):
    """Views into a fused projection, a mask that leaves a block empty, another stream, and a captured call
    replayed on new inputs next to a second captured call."""
    from powershard_b200 import sparse
    from powershard_b200.graphs import GraphedCall
    qkv = rows(23, 1, 700, 3, 4, 128).to(DEV)
    q, k, v = qkv.unbind(2)
    allowed = torch.ones(3, 6, dtype=torch.bool)
    allowed[1] = False
    allowed[2, 3:] = False
    p = sparse.SparseProvider(0.5)
    want = ref_provider(q.cpu(), k.cpu(), v.cpu(), 3, allowed=allowed)
    mask = allowed.to(DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = p(q, k, v, allowed=mask)
    side.synchronize()
    assert_attention(out, *want)
    assert not out[:, 256:512].any()
    first = GraphedCall(p, q, k, v, allowed=mask)
    other = [x.flip(1).contiguous() for x in (q, k, v)]
    second = GraphedCall(p, *other)
    for _ in range(2):  # the two graphs in flight on two streams
        with torch.cuda.stream(side):
            a = first()
        b = second()
        torch.cuda.synchronize()
        assert torch.equal(a, out)
        assert_attention(b, *ref_provider(*(x.cpu() for x in other), 3))
    qkv.copy_(rows(24, 1, 700, 3, 4, 128))
    first()
    torch.cuda.synchronize()
    assert_attention(first.out, *ref_provider(q.cpu(), k.cpu(), v.cpu(), 3, allowed=allowed))


@pytest.mark.gpu
def test_strides_of_axes_of_one(cuda_lib):
    """The stride of an axis with one entry says nothing."""
    from powershard_b200 import sparse
    for lq, heads in ((300, 2), (1, 2), (300, 1), (5, 1)):
        q, k, v = (rows(s, 1, n, heads, 128).to(DEV) for s, n in ((64, lq), (65, 700), (66, 700)))
        odd = []
        for t in (q, k, v):
            st = [3 if n == 1 else s for n, s in zip(t.shape, t.stride())]
            odd.append(t.as_strided(t.shape, st))
            assert odd[-1].is_contiguous()
        p = sparse.SparseProvider(3)
        assert torch.equal(p(*odd), p(q, k, v))
        means = sparse.block_means(k, 128)
        assert torch.equal(sparse.block_means(odd[1], 128), means)
        assert torch.equal(p(*odd, key_means=means), p(q, k, v, key_means=means))
        lists = torch.zeros(1, heads, -(-lq // 256), 1, dtype=torch.int32, device=DEV)
        assert torch.equal(sparse.sparse_attention(*odd, lists), sparse.sparse_attention(q, k, v, lists))


@pytest.mark.gpu
def test_results_do_not_depend_on_what_memory_held(cuda_lib):
    """Two runs give the same bits, with the allocator's blocks full of NaN in between."""
    from powershard_b200 import sparse
    q, k, v = (rows(s, 2, 1300, 3, 128).to(DEV) for s in (25, 26, 27))
    used = lens(1300, 0).to(DEV)
    p = sparse.SparseProvider(4, key_block=64)
    a = p(q, k, v, query_lengths=used, key_lengths=used).clone()
    junk = [torch.full((1 << 24,), float("nan"), device=DEV) for _ in range(4)]
    del junk
    b = p(q, k, v, query_lengths=used, key_lengths=used)
    assert torch.equal(a, b) and not b[1].any()


@pytest.mark.gpu
def test_select_in_several_chunks(cuda_lib):
    """More scores than are held at a time, for a batch with shared key heads."""
    from powershard_b200 import sparse
    g = torch.Generator(device=DEV).manual_seed(31)
    qm = torch.randn(2, 300, 12, 128, device=DEV, generator=g)
    km = torch.randn(2, 4000, 4, 128, device=DEV, generator=g)
    used = lens(4000 * 64 - 3, 77 * 64).to(DEV)
    blocks, counts = sparse.select_blocks(qm, km, 111, key_block=64, key_lengths=used, query_lengths=lens(76800, 70000).to(DEV))
    score = torch.einsum("bqghd,bkgd->bghqk", qm.double().view(2, 300, 4, 3, 128), km.double()).reshape(2, 12, 300, 4000)
    score[1, ..., 77:] = -math.inf
    best = score.sort(dim=-1, descending=True, stable=True).indices[..., :111]
    best[1, ..., 77:] = 4000
    best = best.sort(-1).values
    best[best == 4000] = -1
    best[1, :, -(-70000 // 256):] = -1
    assert torch.equal(blocks.long(), best)
    assert torch.equal(counts.long(), (best >= 0).sum(-1))


@pytest.mark.gpu
def test_offsets_past_32_bits(cuda_lib):
    """Keys and values of more than 2^32 bytes and 2^31 elements: means and attention at their far end."""
    from powershard_b200 import sparse
    n, heads = 1_100_000, 16
    g = torch.Generator(device=DEV).manual_seed(32)
    k, v = (torch.zeros(1, n, heads, 128, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    assert k.numel() > 2 ** 31
    k[:, -5000:].normal_(generator=g)
    v[:, -5000:].normal_(generator=g)
    q = torch.randn(1, 300, heads, 128, dtype=torch.bfloat16, device=DEV, generator=g)
    means = sparse.block_means(k, 128)
    nk = means.shape[1]
    last = ref_means(k[:, (nk - 2) * 128:].cpu(), 128)
    assert ((means[:, -2:].double().cpu() - last).abs() <= 2.0 ** -22).all() and not means[:, :nk - 60].any()
    blocks = torch.tensor([0, nk - 30, nk - 2, nk - 1], dtype=torch.int32).expand(1, heads, 2, 4).contiguous()
    got = sparse.sparse_attention(q, k, v, blocks.to(DEV))
    # the same blocks from a copy without what lies between
    first = n - 5000 - (n - 5000) % 128
    near = lambda x: torch.cat([x[:, :128], x[:, first:]], 1).cpu()  # noqa: E731
    shift = first // 128 - 1
    want, mag = ref_attention(q.cpu(), near(k), near(v), torch.where(blocks > 0, blocks - shift, blocks))
    assert_attention(got, want, mag)


@pytest.mark.gpu
def test_calls_from_two_threads(cuda_lib):
    import threading
    from powershard_b200 import sparse
    p = sparse.SparseProvider(3, key_block=64)
    data = [[rows(40 + 3 * i + j, 1, 900 + 300 * i, 2, 128).to(DEV) for j in range(3)] for i in range(2)]
    alone = [p(*d) for d in data]
    got = [None, None]

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                out = p(*data[i])
            torch.cuda.current_stream().synchronize()
            got[i] = out
    torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert torch.equal(got[0], alone[0]) and torch.equal(got[1], alone[1])
