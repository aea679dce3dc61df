"""Paged key-value cache and one-token attention on the GPU against the
64-bit oracle (oracle/kv_cache_oracle.py).

Slots that no token was written to hold NaN (16 / 32 bits and e4m3) or NaN
scales, so a kernel that lets them in shows.

Tolerances, from the arithmetic the kernels promise (u = 2^-24, fp32):
  score  |ds| <= (D + 8) u a,  a = max_j sm_scale sum_d |q_d k_jd|  (products
         summed in fp32; e4m3 / int8 keys: q is rounded to 11 bits at least
         relative to its largest value, exact for fp16 / bf16 up to 2^-24 of it)
  weight relative 2 |ds| + w,  w = 2^-16 for weights that are fed to the
         tensor cores in 16-bit halves, 2^-20 for fp32 math
  sums   n tokens in lanes of 4 at least, rescaled a tile: (n / 4 + 64) u
  floor  a weight in 16-bit halves may be off by 2^-24 of the row's largest
         weight (fp16 pages) or of its largest weight times scale (codes)
  out    within 2 (2 |ds| + w + sums) sum_j weight_j |v_j|, n floors and half a
         unit of its type
  lse    within |ds| + w + sums + 4 u |lse|
"""
import math

import pytest
import torch

import monarch_attention_b200 as mab
from monarch_attention_b200 import _lib
from oracle import kv_cache_oracle as oracle

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
F32, F16, BF16, E4M3, I8 = (torch.float32, torch.float16, torch.bfloat16, torch.float8_e4m3fn,
                            torch.int8)
CODED = (E4M3, I8)


def blank(shape, dtype):
    """Pages that nothing was written to: NaN where the type has one."""
    if dtype == I8:
        return torch.full(shape, 77, dtype=dtype)
    return torch.full(shape, math.nan, dtype=torch.float32).to(dtype)


def make_cache(g, E, Hk, D, page, lens, dtype, spare=2):
    """CPU pages with lens[e] random tokens a sequence, table (-1 where unused)."""
    per = max(1, max(-(-n // page) for n in lens))
    P = E * per + spare
    ids = torch.randperm(P, generator=g)[: E * per].view(E, per).int()
    table = torch.full((E, per), -1, dtype=torch.int32)
    pages, scales = [blank((P, Hk, page, D), dtype) for _ in range(2)], [None, None]
    if dtype in CODED:
        scales = [torch.full((P, Hk, page), math.nan) for _ in range(2)]
    for e, n in enumerate(lens):
        used = -(-n // page)
        table[e, :used] = ids[e, :used]
    for i in range(2):
        x = torch.randn(E, Hk, max(max(lens), 1), D, generator=g)
        if dtype in CODED:  # tokens of very different sizes
            x = x * torch.exp2(torch.randint(-6, 7, x.shape[:3], generator=g).float())[..., None]
        oracle.write(x, pages[i], scales[i], table, [0] * E, lens)
    return pages[0], pages[1], scales[0], scales[1], table


def run_attend(dev, q, kp, vp, ks, vs, table, lens, mask=None, **kw):
    scales = None if ks is None else (ks.to(dev), vs.to(dev))
    return mab.decode_attention(
        q.to(dev), kp.to(dev), vp.to(dev), table.to(dev),
        torch.tensor(lens, dtype=torch.int32, device=dev), None if mask is None else mask.to(dev),
        scales=scales, return_lse=True, check=True, **kw)


def check_attend(out, lse, ref, q, lens, ct):
    want, want_lse, (mag, wv, pv, pmax_vmax) = ref
    D = q.shape[3]
    ds = (D + 8) * U * mag
    w = 2.0 ** -16 if q.dtype != F32 else 2.0 ** -20
    n = torch.tensor(lens, dtype=torch.float64)[:, None]
    sums = (n / 4 + 64) * U
    tol = (2 * ds + w + sums) * 2 * wv
    if q.dtype != F32:
        tol = tol + n * U * (pmax_vmax if ct == F16 else pv)
    got = out.double().cpu()
    err = (got - want).abs()
    bound = tol[..., None, None] + HALF[q.dtype] * want.abs() + 2.0 ** -25 * (q.dtype == F16)
    assert torch.isfinite(got).all()
    assert (err <= bound).all(), f"max excess {(err - bound).max():.3g}, max err {err.max():.3g}"
    got = lse.double().cpu()
    empty = torch.isinf(want_lse)
    assert (torch.isneginf(got) == empty).all()
    lerr = torch.where(empty, 0.0, (got - want_lse).abs())
    lbound = torch.where(empty, 0.0, ds + w + sums + 4 * U * want_lse.abs())
    assert (lerr <= lbound).all(), f"lse: max excess {(lerr - lbound).max():.3g}"
    assert (out.cpu()[empty] == 0).all()


TYPES = [(F32, F32), (F16, F16), (BF16, BF16), (BF16, E4M3), (F16, E4M3), (F32, E4M3), (BF16, I8),
         (F16, I8), (F32, I8)]
TYPE_IDS = [f"{str(a)[6:]}-{str(b)[6:]}" for a, b in TYPES]
# (E, H, Hk, D, page, lengths)
SHAPES = [
    (1, 1, 1, 64, 16, [1]),
    (3, 12, 12, 64, 16, [0, 1, 33]),                   # an empty sequence beside others
    (4, 4, 4, 128, 16, [31, 32, 33, 64]),              # around a tile's end
    (2, 8, 2, 128, 24, [100, 23]),                     # pages that end inside a tile
    (2, 3, 1, 72, 7, [50, 14]),                        # an odd page, DiT's head size
    (2, 16, 1, 80, 48, [200, 97]),                     # one shared head
    (1, 24, 1, 128, 32, [300]),                        # more query heads than a pass takes
    (1, 40, 2, 64, 64, [130]),
    (2, 2, 1, 256, 16, [70, 3]),
    (1, 9, 1, 256, 8, [65]),
    (2, 10, 2, 96, 1, [40, 39]),                       # pages of one token
    (2, 4, 2, 17, 16, [45, 16]),                       # rows that no vector load fits
    (2, 2, 2, 1, 16, [20, 2]),
    (1, 6, 3, 200, 128, [129]),
    (1, 2, 1, 32, 16, [2000]),                         # one row over many CTAs
    (37, 2, 1, 64, 16, [(7 * i) % 50 for i in range(37)]),
]


@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: f"E{s[0]}H{s[1]}k{s[2]}D{s[3]}p{s[4]}n{max(s[5])}")
@pytest.mark.parametrize("qt,ct", TYPES, ids=TYPE_IDS)
def test_attend(qt, ct, shape, cuda_device):
    E, H, Hk, D, page, lens = shape
    g = torch.Generator().manual_seed(11)
    cache = make_cache(g, E, Hk, D, page, lens, ct)
    q = (2 * torch.randn(E, H, 1, D, generator=g)).to(qt)
    out, lse = run_attend(cuda_device, q, *cache, lens)
    assert out.dtype == qt and out.shape == q.shape
    check_attend(out, lse, oracle.attend(q, *cache, lens), q, lens, ct)


@pytest.mark.parametrize("mt", [torch.bool, torch.uint8, torch.int32, torch.int64, F32, F16, BF16,
                                torch.float64])
@pytest.mark.parametrize("qt,ct", [(F32, F32), (BF16, BF16), (F16, I8)],
                         ids=["f32", "bf16", "f16-int8"])
def test_attend_mask(qt, ct, mt, cuda_device):
    """Masks of every dtype, with holes, rows that they leave empty, and NaN
    and infinities in the tokens that they leave out."""
    E, H, Hk, D, page, lens = 4, 4, 2, 64, 16, [90, 40, 33, 70]
    g = torch.Generator().manual_seed(12)
    kp, vp, ks, vs, table = make_cache(g, E, Hk, D, page, lens, ct)
    keep = torch.rand(E, 96, generator=g) < 0.6
    keep[1] = False
    keep[2, :32] = False  # a whole tile out
    mask = keep.to(mt) if mt == torch.bool else torch.where(keep, 3, 0).to(mt)
    q = torch.randn(E, H, 1, D, generator=g).to(qt)
    ref = oracle.attend(q, kp, vp, ks, vs, table, lens, keep)
    for e, n in enumerate(lens):
        for t in range(n):
            if not keep[e, t]:
                p, s = int(table[e, t // page]), t % page
                if ks is None:
                    kp[p, :, s], vp[p, :, s] = math.nan, -math.inf
                else:
                    ks[p, :, s], vs[p, :, s] = math.inf, math.nan
    out, lse = run_attend(cuda_device, q, kp, vp, ks, vs, table, lens, mask)
    check_attend(out, lse, ref, q, lens, ct)
    # the same mask as a strided view
    wide = torch.zeros(E, 2 * mask.shape[1], dtype=mt)
    wide[:, ::2] = mask
    out2, lse2 = mab.decode_attention(
        q.to(cuda_device), kp.to(cuda_device), vp.to(cuda_device), table.to(cuda_device),
        torch.tensor(lens, dtype=torch.int32, device=cuda_device), wide.to(cuda_device)[:, ::2],
        scales=None if ks is None else (ks.to(cuda_device), vs.to(cuda_device)), return_lse=True)
    assert torch.equal(out, out2) and torch.equal(lse, lse2)


def test_attend_mask_shorter_than_lengths(cuda_device):
    """Positions at and behind the mask's end are out, a mask of no columns leaves nothing."""
    E, H, Hk, D, page, lens = 2, 2, 2, 64, 16, [50, 8]
    g = torch.Generator().manual_seed(13)
    cache = make_cache(g, E, Hk, D, page, lens, BF16)
    q = torch.randn(E, H, 1, D, generator=g).to(BF16)
    mask = torch.ones(E, 20, dtype=torch.bool)
    out, lse = run_attend(cuda_device, q, *cache, lens, mask)
    check_attend(out, lse, oracle.attend(q, *cache, lens, mask), q, lens, BF16)
    out, lse = run_attend(cuda_device, q, *cache, lens, torch.ones(E, 0, dtype=torch.bool))
    assert (out == 0).all() and torch.isneginf(lse).all()


@pytest.mark.parametrize("qt,ct", [(F32, F32), (BF16, BF16), (BF16, E4M3)], ids=["f32", "bf16", "e4m3"])
@pytest.mark.parametrize("E,H,Hk,lens", [
    (1, 8, 1, [40003]),          # one row over every CTA: joined by groups
    (1, 1, 1, [9000]),
    (3, 4, 2, [12001, 5, 7777]),
], ids=["one-row", "one-head", "ragged"])
def test_attend_long(E, H, Hk, lens, qt, ct, cuda_device):
    """Rows that many CTAs share: joined the same way every time, on every
    stream; the oracle's tokens are gathered at once here."""
    D, page = 64, 32
    g = torch.Generator().manual_seed(14)
    per = -(-max(lens) // page)
    table = torch.randperm(E * per, generator=g).view(E, per).int()
    pages, scales, dense = [], [], []
    for _ in range(2):
        x = torch.randn(E * per, Hk, page, D, generator=g)
        c, s = oracle.quantise(x, ct) if ct in CODED else (x.to(ct), None)
        pages.append(c)
        scales.append(s)
        d = c.double() if s is None else c.double() * s.double()[..., None]
        dense.append(d[table.long()].permute(0, 2, 1, 3, 4).reshape(E, Hk, per * page, D))
    q = torch.randn(E, H, 1, D, generator=g).to(qt)
    G = H // Hk
    want = torch.zeros(E, H, 1, D, dtype=torch.float64)
    wl, size = torch.zeros(E, H, dtype=torch.float64), torch.zeros(4, E, H, dtype=torch.float64)
    for e in range(E):
        k, v = (t[e, :, : lens[e]].repeat_interleave(G, 0) for t in dense)
        want[e, :, 0], wl[e], size[:, e] = oracle.attend_dense(q[e].double(), k, v, 1 / math.sqrt(D))
    out, lse = run_attend(cuda_device, q, *pages, *scales, table, lens)
    check_attend(out, lse, (want, wl, size), q, lens, ct)
    args = (q.to(cuda_device), pages[0].to(cuda_device), pages[1].to(cuda_device),
            table.to(cuda_device), torch.tensor(lens, dtype=torch.int32, device=cuda_device))
    kw = dict(scales=None if scales[0] is None else tuple(s.to(cuda_device) for s in scales),
              return_lse=True)
    other = torch.cuda.Stream(cuda_device)
    torch.cuda.synchronize(cuda_device)
    for _ in range(10):
        again = mab.decode_attention(*args, **kw)
        with torch.cuda.stream(other):
            beside = mab.decode_attention(*args, **kw)
        torch.cuda.synchronize(cuda_device)
        for o, l in (again, beside):
            assert torch.equal(o, out) and torch.equal(l, lse)


@pytest.mark.parametrize("layout", ["tokens_first", "padded_rows", "unaligned", "table_columns"])
@pytest.mark.parametrize("qt,ct", [(F32, F32), (F16, F16), (BF16, E4M3)], ids=["f32", "f16", "e4m3"])
def test_attend_strides(qt, ct, layout, cuda_device):
    """Pages, q, out, table and scales as views of other orders and alignments."""
    E, H, Hk, D, page, lens = 3, 4, 2, 64, 16, [60, 17, 2]
    g = torch.Generator().manual_seed(15)
    kp, vp, ks, vs, table = (None if t is None else t.to(cuda_device)
                             for t in make_cache(g, E, Hk, D, page, lens, ct))
    q = torch.randn(E, H, 1, D, generator=g).to(qt).to(cuda_device)
    ln = torch.tensor(lens, dtype=torch.int32, device=cuda_device)
    scales = None if ks is None else (ks, vs)
    want = mab.decode_attention(q, kp, vp, table, ln, scales=scales, return_lse=True, check=True)

    def view(t):
        if layout == "tokens_first":
            return t.transpose(1, 2).contiguous().transpose(1, 2)
        wide = torch.zeros(*t.shape[:3], D + (1 if layout == "unaligned" else 16), dtype=t.dtype,
                           device=t.device)
        wide = wide[..., (1 if layout == "unaligned" else 0):][..., :D]
        wide.copy_(t)
        return wide

    if layout == "table_columns":
        table = table.t().contiguous().t()
        q = q.transpose(0, 1).contiguous().transpose(0, 1)
    else:
        kp, vp = view(kp), view(vp)
        if scales is not None:
            scales = tuple(s.transpose(1, 2).contiguous().transpose(1, 2) for s in scales)
    buf = torch.zeros(E, 1, H * D, dtype=qt, device=cuda_device)
    out = buf.view(E, 1, H, D).permute(0, 2, 1, 3)
    got, lse = mab.decode_attention(q, kp, vp, table, ln, scales=scales, out=out, return_lse=True,
                                    check=True)
    assert got is out
    ref = oracle.attend(q.cpu(), kp.cpu(), vp.cpu(), *(None if s is None else s.cpu() for s in (scales or (None, None))),
                        table.cpu(), lens)
    check_attend(out, lse, ref, q.cpu(), lens, ct)
    assert (out.float() - want[0].float()).abs().max() <= 2 * HALF[qt] * want[0].float().abs().max() + 1e-5


@pytest.mark.parametrize("spread", [1e-6, 1e6])
def test_attend_scale_range(spread, cuda_device):
    """Values whose scales lie far apart: the token that the query picks is
    returned whatever the others' sizes are."""
    E, H, Hk, D, page, n = 1, 1, 1, 64, 16, 64
    g = torch.Generator().manual_seed(16)
    kp, vp = blank((4, Hk, page, D), I8), blank((4, Hk, page, D), I8)
    ks, vs = torch.ones(4, Hk, page), torch.ones(4, Hk, page)
    table = torch.arange(4, dtype=torch.int32)[None]
    x = torch.randn(E, Hk, n, D, generator=g)
    y = torch.randn(E, Hk, n, D, generator=g)
    q = 0.1 * torch.randn(E, H, 1, D, generator=g)
    x[0, 0, 40] = 20 * q[0, 0, 0] / q[0, 0, 0].norm()
    y[0, 0, :] *= spread
    y[0, 0, 40] = torch.randn(D, generator=g)
    oracle.write(x, kp, ks, table, [0], [n])
    oracle.write(y, vp, vs, table, [0], [n])
    q = (40 * q).to(F16)
    out, lse = run_attend(cuda_device, q, kp, vp, ks, vs, table, [n])
    check_attend(out, lse, oracle.attend(q, kp, vp, ks, vs, table, [n]), q, [n], I8)


def test_attend_sm_scale_and_lse_join(cuda_device):
    """Halves of a sequence joined by their lse are the whole."""
    E, H, Hk, D, page, n = 2, 4, 4, 64, 16, 64
    g = torch.Generator().manual_seed(17)
    cache = make_cache(g, E, Hk, D, page, [n] * E, F32)
    q = torch.randn(E, H, 1, D, generator=g)
    out, lse = run_attend(cuda_device, q, *cache, [n] * E, sm_scale=0.3)
    check_attend(out, lse, oracle.attend(q, *cache, [n] * E, sm_scale=0.3), q, [n] * E, F32)
    first = torch.zeros(E, n, dtype=torch.bool)
    first[:, :20] = True
    a, la = run_attend(cuda_device, q, *cache, [n] * E, first, sm_scale=0.3)
    b, lb = run_attend(cuda_device, q, *cache, [n] * E, ~first, sm_scale=0.3)
    l = torch.logaddexp(la, lb)
    joined = a * torch.exp(la - l)[..., None, None] + b * torch.exp(lb - l)[..., None, None]
    assert (joined - out).abs().max() < 1e-5 and (l - lse).abs().max() < 1e-5


def test_attend_in_a_graph(cuda_device):
    """A captured write and attention see the state of each replay."""
    E, H, D, page = 2, 4, 64, 16
    cache = mab.PagedKVCache(8, H, D, max_seqs=E, max_len=64, page_size=page, dtype=BF16,
                             device=cuda_device)
    cache.reserve([64] * E)
    g = torch.Generator(device=cuda_device).manual_seed(18)
    k, v, q = (torch.zeros(E, H, 1, D, dtype=BF16, device=cuda_device) for _ in range(3))

    def step():
        kv_args = (cache.k_pages, cache.v_pages, cache.page_table)
        mab.kv_cache_write(k, v, *kv_args, cache.lengths)
        cache.lengths += 1
        return mab.decode_attention(q, *kv_args, cache.lengths)

    side = torch.cuda.Stream(cuda_device)
    side.wait_stream(torch.cuda.current_stream(cuda_device))
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream(cuda_device).wait_stream(side)
    cache.lengths.zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    cache.lengths.zero_()
    ks, vs = [], []
    for n in range(1, 40):
        for t in (k, v, q):
            t.copy_(torch.randn(t.shape, generator=g, device=cuda_device))
        ks.append(k.clone())
        vs.append(v.clone())
        graph.replay()
        s = torch.einsum("ehqd,ehnd->ehqn", q.double(), torch.cat(ks, 2).double()) / math.sqrt(D)
        want = torch.softmax(s, -1) @ torch.cat(vs, 2).double()
        err = (out.double() - want).abs().max()
        assert err <= 2.0 ** -8 * want.abs().max() + 2.0 ** -15 * 5, n
    mab.check_status(cuda_device)


# ---- store and read back ---------------------------------------------------------------------

PAIRS = [(F32, F32), (F16, F16), (BF16, BF16), (F32, BF16), (BF16, F16), (BF16, E4M3), (F16, E4M3),
         (F32, E4M3), (BF16, I8), (F16, I8), (F32, I8)]


@pytest.mark.parametrize("xt,ct", PAIRS, ids=[f"{str(a)[6:]}-{str(b)[6:]}" for a, b in PAIRS])
@pytest.mark.parametrize("E,Hk,T,D,page,start,count", [
    (1, 1, 1, 64, 16, [0], None),
    (3, 4, 1, 64, 16, [15, 16, 0], None),              # one token, at a page's end and start
    (2, 3, 37, 72, 7, [5, 0], [37, 20]),
    (2, 2, 5, 128, 16, [0, 30], [0, 5]),               # one sequence takes nothing
    (2, 12, 70, 64, 16, [3, 3], [99, -4]),             # counts outside [0, T]
    (1, 2, 9, 256, 4, [1], None),
    (1, 1, 6, 17, 5, [2], None),
    (2, 5, 3, 1, 16, [0, 1], None),
    (1, 3, 33, 200, 8, [0], None),
], ids=lambda x: str(x).replace(" ", ""))
def test_store_and_read(E, Hk, T, D, page, start, count, xt, ct, cuda_device):
    g = torch.Generator().manual_seed(21)
    per = -(-(max(start) + T) // page)
    table = torch.randperm(E * per + 2, generator=g)[: E * per].view(E, per).int()
    shape = (E * per + 2, Hk, page, D)
    x = [(torch.randn(E, T, Hk * D, generator=g) * torch.exp2(
        torch.randint(-12, 12, (E, T, 1), generator=g).float())).to(xt) for _ in range(2)]
    x[0][0, 0] = 0.0  # a token of zeros
    views = [t.view(E, T, Hk, D).permute(0, 2, 1, 3) for t in x]
    took = [T] * E if count is None else [min(max(c, 0), T) for c in count]
    pages = [blank(shape, ct) for _ in range(2)]
    scales = [torch.full(shape[:3], 0.5) if ct in CODED else None for _ in range(2)]
    dp = [p.to(cuda_device) for p in pages]
    ds = None if scales[0] is None else tuple(s.to(cuda_device) for s in scales)
    for t, p, s in zip(views, pages, scales):
        oracle.write(t, p, s, table, start, took)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=cuda_device)
    mab.kv_cache_write(*(t.to(cuda_device) for t in views), *dp, table.to(cuda_device), i32(start),
                       scales=ds, count=None if count is None else i32(count), check=True)
    raw = (lambda t: t.cpu().view(torch.uint8)) if ct.itemsize == 1 else (lambda t: t.cpu())
    for i in range(2):  # every byte: what was written, and what was not
        assert torch.equal(torch.nan_to_num(raw(dp[i]).float(), nan=-7.0),
                           torch.nan_to_num(raw(pages[i]).float(), nan=-7.0))
        if ds is not None:
            assert torch.equal(ds[i].cpu(), scales[i])
    # back as dense tensors
    lens = [s + n for s, n in zip(start, took)]
    for i in range(2):  # positions before start were never written: give them values
        for e in range(E):
            for t in range(start[e]):
                pages[i][int(table[e, t // page]), :, t % page] = torch.ones(Hk, D).to(ct)
    dp = [p.to(cuda_device) for p in pages]
    N = max(1, max(lens) - 1)  # one shorter than the longest
    for dt in (F32, BF16, F16):
        k, v, mask = mab.kv_cache_read(*dp, table.to(cuda_device), i32(lens), N, scales=ds, dtype=dt,
                                       check=True)
        assert k.shape == (E, Hk, N, D) and k.dtype == dt
        for got, p, s in ((k, pages[0], scales[0]), (v, pages[1], scales[1])):
            want = oracle.read(p, s, table, lens, N)
            # a code times its scale is rounded to fp32 and then to the type
            assert torch.equal(got.cpu(), want.float().to(dt))
        assert torch.equal(mask.cpu(), torch.arange(N)[None] < torch.tensor(lens)[:, None])


def test_read_into_strided_out(cuda_device):
    """out= in the (E, N, Hk * D) order of the next projection; the mask and
    tensors are what monarch_attention takes."""
    E, Hk, D, page, lens, N = 2, 4, 64, 16, [128, 100], 128
    g = torch.Generator().manual_seed(22)
    kp, vp, ks, vs, table = make_cache(g, E, Hk, D, page, lens, E4M3)
    bufs = [torch.empty(E, N, Hk * D, dtype=BF16, device=cuda_device) for _ in range(2)]
    out = tuple(b.view(E, N, Hk, D).permute(0, 2, 1, 3) for b in bufs)
    ln = torch.tensor(lens, dtype=torch.int32, device=cuda_device)
    args = (kp.to(cuda_device), vp.to(cuda_device), table.to(cuda_device), ln, N)
    scales = (ks.to(cuda_device), vs.to(cuda_device))
    k, v, mask = mab.kv_cache_read(*args, scales=scales, out=out, check=True)
    k2, v2, _ = mab.kv_cache_read(*args, scales=scales)
    assert torch.equal(k, k2) and torch.equal(v, v2) and k.data_ptr() == bufs[0].data_ptr()
    z = mab.monarch_attention(k, k, v, mask, 2, 16, False, check=True)
    z2 = mab.monarch_attention(k2, k2, v2, mask, 2, 16, False, check=True)
    assert torch.equal(z, z2) and torch.isfinite(z).all()


def test_store_strided_head_dimension(cuda_device):
    """k and v whose head dimension is not the innermost one."""
    E, Hk, T, D, page = 2, 2, 5, 64, 16
    g = torch.Generator().manual_seed(23)
    x = torch.randn(E, Hk, D, T, generator=g).to(BF16).transpose(2, 3)
    table = torch.arange(E, dtype=torch.int32, device=cuda_device)[:, None]
    for ct in (BF16, I8):
        got, want = [], []
        for t in (x, x.contiguous()):
            p = [torch.zeros(E, Hk, page, D, dtype=ct, device=cuda_device) for _ in range(2)]
            s = tuple(torch.zeros(E, Hk, page, device=cuda_device) for _ in range(2)) if ct == I8 else None
            d = t.to(cuda_device)
            assert d.stride() == t.stride()
            mab.kv_cache_write(d, d, *p, table, torch.zeros(E, dtype=torch.int32, device=cuda_device),
                               scales=s, check=True)
            got.append(p[0])
        assert torch.equal(got[0], got[1])


# ---- what does not fit ------------------------------------------------------------------------

def _small(dev, ct=BF16):
    kp, vp = (torch.zeros(4, 2, 16, 64, dtype=ct, device=dev) for _ in range(2))
    table = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32, device=dev)
    return kp, vp, table


@pytest.mark.parametrize("op", ["write", "read", "attend"])
@pytest.mark.parametrize("what,name", [("page", "page that is not there"), ("negative_page", "page that is not there"),
                                       ("length", "beyond its pages"), ("negative", "beyond its pages")])
def test_bad_table_or_length_raises(op, what, name, cuda_device):
    """Device data that does not fit: the kernels leave it out and the call
    raises; the next good call is exact."""
    dev = cuda_device
    kp, vp, table = _small(dev)
    ln = torch.tensor([20, 32], dtype=torch.int32, device=dev)
    good_table, good_ln = table.clone(), ln.clone()
    if what == "page":
        table[1, 1] = 4
    elif what == "negative_page":
        table[0, 1] = -1
    else:
        ln[1] = 33 if what == "length" else -1
    x = torch.ones(2, 2, 1, 64, dtype=BF16, device=dev)

    def go(t, n, check=True):
        if op == "write":
            mab.kv_cache_write(x, x, kp, vp, t, n - 1, check=check)
        elif op == "read":
            mab.kv_cache_read(kp, vp, t, n, 32, check=check)
        else:
            return mab.decode_attention(x, kp, vp, t, n, check=check)

    mab.read_status(dev)
    with pytest.raises(mab.MonarchAttentionError, match=name) as ei:
        go(table, ln + (1 if op == "write" and what == "length" else 0))
    assert ei.value.code == _lib.MA_ERR_DEVICE
    go(good_table, good_ln)
    # without check=True the next call says it
    go(table, ln + (1 if op == "write" and what == "length" else 0), check=False)
    torch.cuda.synchronize(dev)
    with pytest.raises(mab.MonarchAttentionError, match=name):
        mab.decode_attention(x, kp, vp, good_table, good_ln)
    go(good_table, good_ln)


def test_wrong_arguments_are_refused(cuda_device):
    dev = cuda_device
    kp, vp, table = _small(dev)
    ln = torch.tensor([20, 32], dtype=torch.int32, device=dev)
    q = torch.zeros(2, 4, 1, 64, dtype=BF16, device=dev)
    x = torch.zeros(2, 2, 3, 64, dtype=BF16, device=dev)
    e = torch.zeros(4, 2, 16, 64, dtype=E4M3, device=dev)
    sc = torch.zeros(4, 2, 16, device=dev)
    with pytest.raises(ValueError):  # two new tokens
        mab.decode_attention(q.expand(2, 4, 2, 64), kp, vp, table, ln)
    with pytest.raises(ValueError):  # 3 query heads on 2
        mab.decode_attention(q[:, :3], kp, vp, table, ln)
    with pytest.raises(ValueError):
        mab.decode_attention(q[:1], kp, vp, table, ln)
    with pytest.raises(TypeError):
        mab.decode_attention(q.half(), kp, vp, table, ln)
    with pytest.raises(ValueError):  # 64-bit lengths
        mab.decode_attention(q, kp, vp, table, ln.long())
    with pytest.raises(ValueError):
        mab.decode_attention(q, kp, vp, table, ln.cpu())
    with pytest.raises(ValueError):
        mab.decode_attention(q, kp, vp, table.long(), ln)
    with pytest.raises(ValueError):  # codes without scales
        mab.decode_attention(q, e, e, table, ln)
    with pytest.raises(ValueError):  # scales without codes
        mab.decode_attention(q, kp, vp, table, ln, scales=(sc, sc))
    with pytest.raises(ValueError):
        mab.decode_attention(q, e, e, table, ln, scales=(sc[:3], sc))
    with pytest.raises(ValueError):
        mab.decode_attention(q, kp, vp[..., :32], table, ln)
    with pytest.raises(ValueError):  # head dimension not innermost
        mab.decode_attention(q, kp.transpose(2, 3).contiguous().transpose(2, 3), vp, table, ln)
    with pytest.raises(ValueError):
        mab.decode_attention(q, kp, vp, table, ln, torch.ones(3, 32, device=dev))
    with pytest.raises(mab.MonarchAttentionError):
        mab.decode_attention(q, kp, vp, table, ln, sm_scale=0.0)
    with pytest.raises(RuntimeError):
        mab.decode_attention(q.clone().requires_grad_(), kp, vp, table, ln)
    with pytest.raises(TypeError):
        mab.kv_cache_write(x.double(), x.double(), kp, vp, table, ln)
    with pytest.raises(ValueError):
        mab.kv_cache_write(x[:, :1], x[:, :1], kp, vp, table, ln)
    with pytest.raises(ValueError):
        mab.kv_cache_write(x, x, kp, vp, table, ln, count=ln[:1])
    with pytest.raises(ValueError):
        mab.kv_cache_read(kp, vp, table, ln, -1)
    with pytest.raises(TypeError):
        mab.kv_cache_read(kp, vp, table, ln, 4, dtype=torch.float64)
    big = torch.zeros(1, 1, 1, 257, dtype=BF16, device=dev)
    with pytest.raises(mab.MonarchAttentionError):  # head dim above 256
        mab.kv_cache_read(big, big, table[:, :1], ln, 1)
    # nothing to do
    none = table[:0]
    assert mab.decode_attention(q[:0], kp, vp, none, ln[:0]).shape == (0, 4, 1, 64)
    mab.kv_cache_write(x[:, :, :0], x[:, :, :0], kp, vp, table, ln)
    assert mab.kv_cache_read(kp, vp, table, ln, 0)[0].shape == (2, 2, 0, 64)
    mab.check_status(dev)


# ---- the cache object --------------------------------------------------------------------------

@pytest.mark.parametrize("ct,D", [(BF16, 64), (F16, 72), (E4M3, 72), (I8, 64), (F32, 40)])
def test_cache_object_grows_and_frees(ct, D, cuda_device):
    E, H, Hk, page = 3, 4, 2, 16
    dt = ct if ct not in CODED else BF16
    g = torch.Generator().manual_seed(24)
    cache = mab.PagedKVCache(14, Hk, D, max_seqs=E, max_len=80, page_size=page, dtype=ct,
                             device=cuda_device)
    ks, vs = [], []
    for T in (17, 1, 1, 13, 1):
        k, v = (torch.randn(E, Hk, T, D, generator=g).to(dt) for _ in range(2))
        cache.append(k.to(cuda_device), v.to(cuda_device), check=True)
        ks.append(k)
        vs.append(v)
    k, v = torch.cat(ks, 2), torch.cat(vs, 2)
    assert cache.lengths.tolist() == [33] * E and cache.free_pages == 14 - 9
    gk, gv, mask = cache.read(dtype=F32)
    assert mask.all() and mask.shape == (E, 33)
    for got, x in ((gk, k), (gv, v)):
        if ct in CODED:
            c, s = oracle.quantise(x, ct)
            x = (c.double() * s.double()[..., None]).float()
        assert torch.equal(got.cpu(), x.float())
    q = torch.randn(E, H, 1, D, generator=g).to(dt)
    out = cache.attend(q.to(cuda_device), check=True)
    s = (q.double().view(E, Hk, 2, D) @ gk.cpu().double().transpose(2, 3)) / math.sqrt(D)
    want = (torch.softmax(s, -1) @ gv.cpu().double()).view(E, H, 1, D)
    assert (out.cpu().double() - want).abs().max() <= (HALF[dt] + 2.0 ** -15) * 4
    with pytest.raises(RuntimeError, match="full"):
        cache.reserve([80, 80, 80])
    with pytest.raises(ValueError, match="max_len"):
        cache.reserve([81, 0, 0])
    cache.free(1)
    assert cache.free_pages == 14 - 6 and cache.lengths.tolist() == [33, 0, 33]
    out2 = cache.attend(q.to(cuda_device), check=True)
    assert (out2[1] == 0).all() and torch.equal(out2[0], out[0]) and torch.equal(out2[2], out[2])
    # a ragged append: sequence 1 starts again, 2 takes nothing
    k, v = (torch.randn(E, Hk, 4, D, generator=g).to(dt).to(cuda_device) for _ in range(2))
    cache.append(k, v, count=torch.tensor([2, 4, 0], dtype=torch.int32, device=cuda_device), check=True)
    assert cache.lengths.tolist() == [35, 4, 33]


# ---- blocks of memory, many rows, long caches -----------------------------------------------------

@pytest.mark.parametrize("masked", [False, True], ids=["", "mask"])
@pytest.mark.parametrize("H,Hk", [(1, 1), (4, 1), (10, 2), (16, 2), (24, 2), (40, 2)])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("qt,ct", [(F16, F16), (BF16, BF16), (BF16, E4M3), (F16, I8)],
                         ids=["f16", "bf16", "e4m3", "int8"])
def test_attend_block_tiles(qt, ct, D, H, Hk, masked, cuda_device):
    """Pages of whole tiles: a tile is one block of memory, full or in part, of
    every group of query heads; NaN where nothing is valid."""
    E, page, lens = 3, 32, [100, 33, 64]
    g = torch.Generator().manual_seed(31 + H)
    kp, vp, ks, vs, table = make_cache(g, E, Hk, D, page, lens, ct)
    q = torch.randn(E, H, 1, D, generator=g).to(qt)
    keep = None
    if masked:
        keep = torch.rand(E, 100, generator=g) < 0.8
        keep[2, 32:] = False
    ref = oracle.attend(q, kp, vp, ks, vs, table, lens, keep)
    if masked:
        for e, n in enumerate(lens):
            for t in range(n):
                if not keep[e, t]:
                    p, s = int(table[e, t // page]), t % page
                    if ks is None:
                        kp[p, :, s], vp[p, :, s] = math.inf, math.nan
                    else:
                        ks[p, :, s], vs[p, :, s] = math.nan, math.inf
    out, lse = run_attend(cuda_device, q, kp, vp, ks, vs, table, lens, keep)
    check_attend(out, lse, ref, q, lens, ct)


@pytest.mark.parametrize("E,Hk,most", [(64, 3, 70), (70, 2, 40), (130, 8, 90), (700, 1, 9), (9, 70, 40)])
@pytest.mark.parametrize("qt,ct", [(F32, F32), (BF16, BF16)], ids=["f32", "bf16"])
def test_attend_many_rows(qt, ct, E, Hk, most, cuda_device):
    """More sequences than a warp's lanes or a CTA's threads, more rows than CTAs,
    empty sequences among them, one long one."""
    D, page = 32, 16
    g = torch.Generator().manual_seed(32)
    lens = torch.randint(0, most, (E,), generator=g)
    lens[E // 2] = 4 * most
    per = -(-int(lens.max()) // page)
    table = torch.randperm(E * per, generator=g).view(E, per).int()
    kp, vp = (torch.randn(E * per, Hk, page, D, generator=g).to(ct) for _ in range(2))
    q = torch.randn(E, Hk, 1, D, generator=g).to(qt)
    want = torch.zeros(E, Hk, 1, D, dtype=torch.float64)
    wl = torch.full((E, Hk), -math.inf, dtype=torch.float64)
    size = torch.zeros(4, E, Hk, dtype=torch.float64)
    for e, n in enumerate(lens.tolist()):
        if n:
            k, v = (t.double()[table[e].long()].transpose(0, 1).reshape(Hk, -1, D)[:, :n] for t in (kp, vp))
            want[e, :, 0], wl[e], size[:, e] = oracle.attend_dense(q[e].double(), k, v, 1 / math.sqrt(D))
    out, lse = run_attend(cuda_device, q, kp, vp, None, None, table, lens.tolist())
    check_attend(out, lse, (want, wl, size), q, lens.tolist(), ct)


def test_attend_page_table_for_very_long_sequences(cuda_device):
    """A table whose longest sequences would give more tiles than 32-bit sums hold."""
    E, Hk, D, page, lens = 2, 32, 64, 64, [100, 3]
    g = torch.Generator().manual_seed(33)
    cache = list(make_cache(g, E, Hk, D, page, lens, BF16))
    table = torch.full((E, 1 << 22), -1, dtype=torch.int32)
    table[:, : cache[4].shape[1]] = cache[4]
    q = torch.randn(E, Hk, 1, D, generator=g).to(BF16)
    small = run_attend(cuda_device, q, *cache, lens)
    cache[4] = table
    wide = run_attend(cuda_device, q, *cache, lens)
    check_attend(*small, oracle.attend(q, *cache[:4], table, lens), q, lens, BF16)
    check_attend(*wide, oracle.attend(q, *cache[:4], table, lens), q, lens, BF16)


@pytest.mark.parametrize("ct,page", [(I8, 16), (I8, 32), (BF16, 32), (F32, 16)],
                         ids=["int8", "int8-blocks", "bf16", "f32"])
def test_offsets_beyond_32_bits(ct, page, cuda_device):
    """Pages behind the first 2^31 elements (and 2^32 bytes): stored, read back and
    attended to as in a small cache, bit for bit."""
    dev, Hk, D, n = cuda_device, 8, 128, 50
    dt = BF16 if ct == I8 else ct
    P = (1 << 31) // (Hk * page * D) + 8
    g = torch.Generator(device=dev).manual_seed(34)
    k, v = (torch.randn(1, Hk, n, D, generator=g, device=dev).to(dt) for _ in range(2))
    q = torch.randn(1, 2 * Hk, 1, D, generator=g, device=dev).to(dt)
    per = -(-n // page)
    ln = torch.tensor([n], dtype=torch.int32, device=dev)
    got = []
    for pages, first in ((P, P - per), (per + 1, 1)):
        kp, vp = (torch.empty(pages, Hk, page, D, dtype=ct, device=dev) for _ in range(2))
        scales = None
        if ct == I8:
            scales = tuple(torch.empty(pages, Hk, page, device=dev) for _ in range(2))
        table = torch.arange(first, first + per, dtype=torch.int32, device=dev)[None]
        mab.kv_cache_write(k, v, kp, vp, table, torch.zeros_like(ln), scales=scales, check=True)
        back = mab.kv_cache_read(kp, vp, table, ln, n, scales=scales, check=True)
        got.append((*back, *mab.decode_attention(q, kp, vp, table, ln, scales=scales, return_lse=True,
                                                 check=True)))
        del kp, vp, scales
        torch.cuda.empty_cache()
    assert (P - per) * Hk * page * D > (1 << 31) - (1 << 24)
    for a, b in zip(*got):
        assert torch.equal(a, b)
    assert torch.isfinite(got[0][3]).all() and got[0][2].all()


@pytest.mark.parametrize("ct", [F16, BF16, E4M3, I8, F32])
def test_attend_unaligned_q_and_out(ct, cuda_device):
    """q and out that start between the boundaries that wide loads and stores need."""
    E, H, Hk, D, page, lens = 2, 8, 2, 64, 32, [70, 40]
    dt = ct if ct not in CODED else F16
    g = torch.Generator().manual_seed(35)
    cache = make_cache(g, E, Hk, D, page, lens, ct)
    q = torch.randn(E, H, 1, D, generator=g).to(dt)
    ref = oracle.attend(q, *cache, lens)
    wide = torch.zeros(E, H, 1, D + 3, dtype=dt, device=cuda_device)
    qv, buf = wide[..., 1:D + 1], torch.full_like(wide, 7.0)
    qv.copy_(q)
    out = buf[..., 3:]
    scales = None if cache[2] is None else (cache[2].to(cuda_device), cache[3].to(cuda_device))
    _, lse = mab.decode_attention(qv, cache[0].to(cuda_device), cache[1].to(cuda_device),
                                  cache[4].to(cuda_device),
                                  torch.tensor(lens, dtype=torch.int32, device=cuda_device),
                                  scales=scales, out=out, return_lse=True, check=True)
    check_attend(out, lse, ref, q, lens, ct)
    assert (buf[..., :3] == 7).all()


@pytest.mark.parametrize("ct", [E4M3, I8])
def test_store_infinity_and_nan(ct, cuda_device):
    """A token with an infinity or NaN has an infinite or NaN scale, and no other
    token changes."""
    dev, D = cuda_device, 64
    x = torch.ones(1, 1, 4, D, dtype=BF16)
    x[0, 0, 1, 5], x[0, 0, 2, 60] = math.inf, math.nan
    p = [torch.zeros(1, 1, 16, D, dtype=ct, device=dev) for _ in range(2)]
    s = tuple(torch.zeros(1, 1, 16, device=dev) for _ in range(2))
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)
    mab.kv_cache_write(x.to(dev), x.to(dev), *p, i32([[0]]), i32([0]), scales=s, check=True)
    for sc in s:
        assert torch.isinf(sc[0, 0, 1]) and torch.isnan(sc[0, 0, 2])
        assert torch.isfinite(sc[0, 0, [0, 3]]).all()
    k, v, _ = mab.kv_cache_read(*p, i32([[0]]), i32([4]), 4, scales=s, dtype=F32, check=True)
    for t in (k, v):
        # the scale's fp32 rounding and the code's half step
        assert ((t[0, 0, [0, 3]] - 1).abs() <= 2.0 ** -4).all()
        assert not torch.isfinite(t[0, 0, 1, 5]) and torch.isnan(t[0, 0, 2]).all()


@pytest.mark.parametrize("size", [1.0, 40.0], ids=["", "steep"])
@pytest.mark.parametrize("H,Hk", [(2, 2), (4, 2), (3, 1), (8, 2), (5, 1), (24, 1)])
@pytest.mark.parametrize("D", [60, 64, 72, 128, 200, 256])
@pytest.mark.parametrize("ct", [F32, E4M3, I8], ids=["f32", "e4m3", "int8"])
def test_attend_shared_heads_fp32(ct, D, H, Hk, size, cuda_device):
    """Passes of one and four heads in 32 bits, a pass partly filled; tokens that are not
    valid beside ones that are, with NaN and infinity behind them; scores whose running
    maximum moves often (steep) and by less than a weight's room."""
    E, page, lens = 4, 24, [131, 0, 1, 66]
    g = torch.Generator().manual_seed(41 + H)
    kp, vp, ks, vs, table = make_cache(g, E, Hk, D, page, lens, ct)
    q = torch.randn(E, H, 1, D, generator=g) * size
    keep = torch.rand(E, 131, generator=g) < 0.7
    keep[2, 0] = True
    keep[3, 5:40] = False
    ref = oracle.attend(q, kp, vp, ks, vs, table, lens, keep)
    for e, n in enumerate(lens):
        for t in range(n):
            if not keep[e, t]:
                at = int(table[e, t // page]), slice(None), t % page
                if ks is None:
                    kp[at], vp[at] = math.nan, math.inf
                else:
                    ks[at], vs[at] = math.inf, math.nan
    out, lse = run_attend(cuda_device, q, kp, vp, ks, vs, table, lens, keep)
    check_attend(out, lse, ref, q, lens, ct)
