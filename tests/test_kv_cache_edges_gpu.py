"""Paged key-value cache and one-token attention where they can go wrong: scores that are
not numbers, rows whose weights lie far apart, page entries that a mask leaves out, what the
cache object promises of its host side.

Wanted values are computed in 64 bits.  u = 2^-24 (fp32); half a unit of a result's type is
2^-11 (fp16) or 2^-8 (bf16, which includes one flipped last bit) of it.
"""
import math

import pytest
import torch

import monarch_attention_b200 as mab

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
F32, F16, BF16, E4M3, I8 = (torch.float32, torch.float16, torch.bfloat16, torch.float8_e4m3fn,
                            torch.int8)
CODED = {E4M3: 448.0, I8: 127.0}
HALF = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}
TYPES = [(F32, F32), (F16, F16), (BF16, BF16), (BF16, E4M3), (F16, E4M3), (F32, E4M3), (BF16, I8),
         (F16, I8), (F32, I8)]
TYPE_IDS = [f"{str(a)[6:]}-{str(b)[6:]}" for a, b in TYPES]


def i32(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def paged(x, ct, page, width, dev):
    """x (E, Hk, n, D) in 64 bits -> pages, scales, page table of `width` columns, and the
    values that the pages hold, in 64 bits."""
    E, Hk, n, D = x.shape
    per = -(-n // page)
    pad = torch.zeros(E, Hk, per * page, D, dtype=torch.float64, device=dev)
    pad[:, :, :n] = x
    rows = pad.view(E, Hk, per, page, D).permute(0, 2, 1, 3, 4).reshape(E * per, Hk, page, D)
    scale = None
    if ct in CODED:
        scale = (rows.float().abs().amax(-1).clamp_min(1e-12) / CODED[ct])
        code = rows.float() / scale[..., None]
        pages = code.round().to(ct) if ct == I8 else code.to(ct)
        held = pages.double() * scale.double()[..., None]
    else:
        pages = rows.to(ct)
        held = pages.double()
    table = torch.full((E, max(width, per)), -1, dtype=torch.int32, device=dev)
    table[:, :per] = torch.arange(E * per, device=dev).view(E, per)
    held = held.view(E, per, Hk, page, D).permute(0, 2, 1, 3, 4).reshape(E, Hk, per * page, D)[:, :, :n]
    return pages, scale, table, held


def dense(q, k, v, sm_scale):
    """out (E, H, 1, D) and lse (E, H) in 64 bits of q (E, H, 1, D), k, v (E, Hk, n, D)."""
    E, H, _, D = q.shape
    s = (q.double().view(E, k.shape[1], -1, D) @ k.transpose(2, 3)) * sm_scale
    return (torch.softmax(s, -1) @ v).view(E, H, 1, D), torch.logsumexp(s, -1).view(E, H)


# ---- scores that are not numbers ------------------------------------------------------------------

# (head dim, page size, columns of the page table, query heads, kv heads): a row taken whole, rows
# cut into pieces, tiles that are blocks of memory and others, passes of one to sixteen heads
NAN_SHAPES = [(64, 16, 0, 4, 2), (64, 32, 400, 2, 2), (128, 32, 400, 16, 2), (128, 24, 400, 24, 2),
              (256, 32, 0, 6, 2)]


@pytest.mark.parametrize("D,page,width,H,Hk", NAN_SHAPES)
@pytest.mark.parametrize("qt,ct", TYPES, ids=TYPE_IDS)
@pytest.mark.parametrize("what", ["query", "query_infinities", "only_key", "key_alone_in_its_tile",
                                  "tile_of_keys"])
def test_nan_scores_are_not_left_out(what, qt, ct, D, page, width, H, Hk, cuda_device):
    """A token that is valid counts whatever its score is: a NaN among a row's scores makes
    its result and lse NaN, wherever the work was cut; the other rows stay as they are."""
    dev = cuda_device
    g = torch.Generator(device=dev).manual_seed(51)
    E = 2
    n = {"only_key": 1, "key_alone_in_its_tile": 33, "tile_of_keys": 3000}.get(what, 70)
    if width == 0 and n > 2000:
        n = 1500  # a row that still goes to one CTA in 16 bits
    k, v = (torch.randn(E, Hk, n, D, generator=g, device=dev, dtype=torch.float64) for _ in range(2))
    kp, ks, table, kd = paged(k, ct, page, width, dev)
    vp, vs, _, vd = paged(v, ct, page, width, dev)
    q = torch.randn(E, H, 1, D, generator=g, device=dev).to(qt)
    want, want_lse = dense(q, kd, vd, 1 / math.sqrt(D))
    bad = torch.zeros(E, H, dtype=torch.bool, device=dev)
    if what == "query":
        q[1, 1, 0, 3] = math.nan
        bad[1, 1] = True
    elif what == "query_infinities":
        q[1, 1, 0, 3], q[1, 1, 0, 5] = math.inf, -math.inf
        bad[1, 1] = True
        # so that every score is infinity - infinity
        kp[..., 3] = kp[..., 5] = torch.ones((), dtype=F32, device=dev).to(ct)
        held = torch.ones(E, Hk, n, device=dev, dtype=torch.float64)
        if ks is not None:
            per = -(-n // page)
            held = ks.double().view(E, per, Hk, page).permute(0, 2, 1, 3).reshape(E, Hk, -1)[:, :, :n]
        kd[..., 3] = kd[..., 5] = held
        ok = q.clone()
        ok[1, 1] = 0
        want, want_lse = dense(ok, kd, vd, 1 / math.sqrt(D))
    else:
        first, last = {"only_key": (0, 1), "key_alone_in_its_tile": (32, 33),
                       "tile_of_keys": (1024, 1056)}[what]
        for t in range(first, last):
            at = int(table[1, t // page]), 1, t % page
            if ks is None:
                kp[at][2] = math.nan
            else:
                ks[at] = math.nan
        bad[1, H // Hk:] = True
    out, lse = mab.decode_attention(q, kp, vp, table, i32([n] * E, dev), return_lse=True, check=True,
                                    scales=None if ks is None else (ks, vs))
    assert torch.isnan(out[bad]).all() and torch.isnan(lse[bad]).all()
    assert torch.isfinite(out[~bad]).all()
    # the others: scores summed in fp32, a half unit of the result, weights of 16 bits
    err = (out.double() - want)[~bad].abs().max()
    assert err <= (HALF[qt] + 2.0 ** -14) * 4, float(err)
    assert (lse.double() - want_lse)[~bad].abs().max() <= 1e-4

@pytest.mark.parametrize("D,page,width,H,Hk", NAN_SHAPES)
@pytest.mark.parametrize("ct", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
def test_scores_of_minus_infinity_weigh_nothing(ct, D, page, width, H, Hk, cuda_device):
    """Beside others, as if they were not there; alone, as a row without a token."""
    dev, E, n = cuda_device, 2, 130
    g = torch.Generator(device=dev).manual_seed(60)
    k, v = (torch.randn(E, Hk, n, D, generator=g, device=dev, dtype=torch.float64) for _ in range(2))
    kp, _, table, kd = paged(k, ct, page, width, dev)
    vp, _, _, vd = paged(v, ct, page, width, dev)
    q = torch.randn(E, H, 1, D, generator=g, device=dev).to(ct)
    q[..., 3] = 1
    for t in range(n):
        if t not in (40, 41, 100):
            kp[int(table[1, t // page]), :, t % page, 3] = -math.inf
        kp[int(table[0, t // page]), :, t % page, 3] = -math.inf
    out, lse = mab.decode_attention(q, kp, vp, table, i32([n] * E, dev), return_lse=True, check=True)
    at = torch.tensor([40, 41, 100], device=dev)
    want, want_lse = dense(q[1:], kd[1:, :, at], vd[1:, :, at], 1 / math.sqrt(D))
    assert (out[0] == 0).all() and torch.isneginf(lse[0]).all()
    assert (out[1:].double() - want).abs().max() <= (HALF[ct] + 2.0 ** -14) * 4
    assert (lse[1:].double() - want_lse).abs().max() <= 1e-4


# ---- rows whose weights lie far apart ---------------------------------------------------------------

def _sink(ct, qt, H, Hk, D, page, n, nats, where, sink_value, dev, E=1):
    """One token scores `nats` above all others: q is 8 in one dimension, where the others'
    keys are 0.  Values have one sign, so no error cancels.  E sequences share the pages."""
    g = torch.Generator(device=dev).manual_seed(52)
    k = torch.zeros(1, Hk, n, D, dtype=torch.float64, device=dev)
    k[:, :, where, 0] = nats * math.sqrt(D) / 8
    v = 512 * (1 + torch.rand(1, Hk, n, D, generator=g, device=dev, dtype=torch.float64))
    if sink_value == 0:
        v[:, :, where] = 0
    kp, ks, table, kd = paged(k, ct, page, 0, dev)
    vp, vs, _, vd = paged(v, ct, page, 0, dev)
    q = torch.zeros(1, H, 1, D, dtype=qt, device=dev)
    q[..., 0] = 8
    out, lse = mab.decode_attention(q.expand(E, -1, -1, -1), kp, vp, table.expand(E, -1),
                                    i32([n] * E, dev), return_lse=True, check=True,
                                    scales=None if ks is None else (ks, vs))
    want, want_lse = dense(q, kd, vd, 1 / math.sqrt(D))
    return out, lse, want, want_lse, vd


# (sequences, tokens, nats, the large token): rows taken whole, cut over many CTAs, a CTA each
SINKS = [(1, 24, 14.0, 0), (1, 24, 17.5, 0), (1, 1024, 16.0, 3), (1, 1024, 20.0, 1023),
         (1, 65536, 17.5, 0), (600, 9000, 17.0, 4000)]


@pytest.mark.parametrize("E,n,nats,where", SINKS)
@pytest.mark.parametrize("H,Hk,D,page", [(2, 2, 64, 32), (4, 1, 64, 16), (8, 1, 128, 32), (24, 1, 80, 16),
                                         (16, 1, 128, 32), (8, 1, 256, 32), (3, 1, 256, 16)])
def test_small_weights_of_fp16_pages_count(H, Hk, D, page, E, n, nats, where, cuda_device):
    """Many small weights beside a large one of a token that holds 0: the small ones are the
    result.  Scores are right to (D + 8) u of their size (plus a unit each of their product with
    log2 e and of their difference from the maximum), weights to 2^-16 of theirs and 2^-44 of the
    largest, sums of n to (n / 4 + 64) u."""
    out, lse, want, want_lse, vd = _sink(F16, F16, H, Hk, D, page, n, nats, where, 0, cuda_device, E)
    rel = 2 * (D + 8) * U * nats + 2.0 ** -16 + (n / 4 + 64) * U
    tol = (2 * rel + HALF[F16]) * want.abs() + n * 2.0 ** -44 * vd.abs().max()
    err = (out.double() - want).abs()
    assert (want > 2.0 ** -12).all()  # in fp16's normal range
    assert (err <= tol).all(), f"{float((err / want).max()):.3g} of the result"
    assert (lse.double() - want_lse).abs().max() <= rel + 4 * U * nats


@pytest.mark.parametrize("ct", [E4M3, I8], ids=["e4m3", "int8"])
@pytest.mark.parametrize("H,D,page", [(1, 64, 32), (4, 80, 16), (8, 128, 32), (16, 64, 16), (5, 256, 32)])
def test_small_weights_of_coded_pages_count(H, D, page, ct, cuda_device):
    """2^19 weights just below 2^-25 beside one of 1: together they are 1.5 % of the result, a
    warp's quarter of them 0.36 %.  600 sequences, so that a CTA has about a row.  What sums
    of a warp's quarter may lose in fp32, 16 tokens at a time in two halves, each sum off by up to
    2^-23: n 2^-28; weights' floor n 2^-33 of the largest product of weight and value."""
    n, nats = 1 << 19, 17.4
    out, lse, want, want_lse, vd = _sink(ct, F16, H, 1, D, page, n, nats, 7, 1, cuda_device, 600)
    tail = math.exp(math.log(n) - nats)
    rel = 2 * (D + 8) * U * nats + 2.0 ** -16
    tol = (2 * rel * tail + n * (2.0 ** -28 + 2.0 ** -33)) * vd.abs().max() + HALF[F16] * want.abs()
    err = (out.double() - want).abs()
    assert (err <= tol).all(), f"{float((err / want).max()):.3g} of the result"
    assert (lse.double() - want_lse).abs().max() <= rel + n * 2.0 ** -28 + 4 * U * nats

# ---- page entries that a mask leaves out --------------------------------------------------------------

@pytest.mark.parametrize("qt,ct", TYPES, ids=TYPE_IDS)
@pytest.mark.parametrize("page", [16, 32])
def test_pages_of_masked_tokens_may_be_gone(page, qt, ct, cuda_device):
    """Entries of pages that were given back (-1) or never were (num_pages) under a mask's
    zeros, and behind its end, are not used: no failure is reported."""
    dev, E, H, Hk, D, n = cuda_device, 2, 4, 2, 64, 200
    g = torch.Generator(device=dev).manual_seed(53)
    k, v = (torch.randn(E, Hk, n, D, generator=g, device=dev, dtype=torch.float64) for _ in range(2))
    kp, ks, table, kd = paged(k, ct, page, 0, dev)
    vp, vs, _, vd = paged(v, ct, page, 0, dev)
    q = torch.randn(E, H, 1, D, generator=g, device=dev).to(qt)
    mask = torch.zeros(E, 5 * 32, dtype=torch.bool, device=dev)
    mask[0, 64:130], mask[1, 32:96] = True, True
    mask[0, 70:75] = False
    want, want_lse = [], []
    for e in range(E):
        at = mask[e].nonzero()[:, 0]
        o, l = dense(q[e:e + 1], kd[e:e + 1, :, at], vd[e:e + 1, :, at], 1 / math.sqrt(D))
        want.append(o)
        want_lse.append(l)
    table[0, : 64 // page], table[0, 160 // page:] = -1, kp.shape[0]
    table[1, : 32 // page], table[1, 96 // page:] = kp.shape[0], -1
    for _ in range(2):  # the second call would raise what the first one reported
        out, lse = mab.decode_attention(q, kp, vp, table, i32([n] * E, dev), mask, return_lse=True,
                                        scales=None if ks is None else (ks, vs))
    mab.check_status(dev)
    assert (out.double() - torch.cat(want)).abs().max() <= (HALF[qt] + 2.0 ** -14) * 4
    assert (lse.double() - torch.cat(want_lse)).abs().max() <= 1e-4


@pytest.mark.parametrize("qt,ct", [(F32, F32), (BF16, BF16), (F16, I8)], ids=["f32", "bf16", "int8"])
def test_missing_page_of_a_valid_token_is_reported(qt, ct, cuda_device):
    """The same entries under valid tokens: reported, and the tokens left out."""
    dev, E, H, Hk, D, page, n = cuda_device, 1, 2, 2, 64, 32, 96
    g = torch.Generator(device=dev).manual_seed(54)
    k, v = (torch.randn(E, Hk, n, D, generator=g, device=dev, dtype=torch.float64) for _ in range(2))
    kp, ks, table, kd = paged(k, ct, page, 0, dev)
    vp, vs, _, vd = paged(v, ct, page, 0, dev)
    q = torch.randn(E, H, 1, D, generator=g, device=dev).to(qt)
    table[0, 1] = -1
    at = torch.cat([torch.arange(32, device=dev), torch.arange(64, 96, device=dev)])
    want, _ = dense(q, kd[:, :, at], vd[:, :, at], 1 / math.sqrt(D))
    out = mab.decode_attention(q, kp, vp, table, i32([n], dev), torch.ones(E, n, device=dev),
                               scales=None if ks is None else (ks, vs))
    with pytest.raises(mab.MonarchAttentionError, match="page that is not there"):
        mab.check_status(dev)
    assert (out.double() - want).abs().max() <= (HALF[qt] + 2.0 ** -14) * 4

# ---- a query whose elements differ in size, with codes ------------------------------------------------

@pytest.mark.parametrize("qt", [BF16, F16])
@pytest.mark.parametrize("ct", [E4M3, I8], ids=["e4m3", "int8"])
@pytest.mark.parametrize("H,D,page", [(1, 64, 32), (8, 128, 16), (24, 80, 32)])
def test_small_elements_of_a_query_count(H, D, page, ct, qt, cuda_device):
    """A channel of q that is far larger than the others and meets keys of 0: the others
    decide.  They lie 2^24 below it and are to count in full: scores are right to (D + 8) u
    of their size, and what 16-bit elements lose is 2^-39 of the largest one's."""
    dev, n = cuda_device, 150
    g = torch.Generator(device=dev).manual_seed(55)
    k, v = (torch.randn(1, 1, n, D, generator=g, device=dev, dtype=torch.float64) for _ in range(2))
    k[..., 7] = 0
    kp, ks, table, kd = paged(k, ct, page, 0, dev)
    vp, vs, _, vd = paged(v, ct, page, 0, dev)
    big = 2.0 ** 22 if qt == BF16 else 2.0 ** 14
    q = torch.randn(1, H, 1, D, generator=g, device=dev) * big * 2.0 ** -24
    q[..., 7] = big
    q = q.to(qt)
    scale = 2.0 ** 24 / big / math.sqrt(D)
    want, want_lse = dense(q, kd, vd, scale)
    out, lse = mab.decode_attention(q, kp, vp, table, i32([n], dev), return_lse=True, check=True,
                                    scales=(ks, vs), sm_scale=scale)
    mag = (q.double().abs() @ kd.abs().repeat_interleave(H, 1).transpose(2, 3)).amax() * scale
    ds = float(mag) * (D + 8) * U + D * 2.0 ** -39 * 2.0 ** 24 * float(kd.abs().max()) / math.sqrt(D)
    assert (lse.double() - want_lse).abs().max() <= ds + 2.0 ** -16 + 70 * U + 4 * U * want_lse.abs().max()
    tol = 2 * (2 * ds + 2.0 ** -16 + 120 * U) * vd.abs().max() + HALF[qt] * want.abs()
    assert ((out.double() - want).abs() <= tol).all()

# ---- the host's side ------------------------------------------------------------------------------------

def test_read_back_refuses_another_shape_of_out(cuda_device):
    dev = cuda_device
    kp, vp = (torch.zeros(4, 2, 16, 64, dtype=BF16, device=dev) for _ in range(2))
    table, ln = i32([[0, 1], [2, 3]], dev), i32([20, 32], dev)
    out = tuple(torch.zeros(2, 2, 31, 64, dtype=BF16, device=dev) for _ in range(2))
    with pytest.raises(ValueError, match=r"\(2, 2, 32, 64\); got \(2, 2, 31, 64\)"):
        mab.kv_cache_read(kp, vp, table, ln, 32, out=out)


@pytest.mark.parametrize("which", ["k", "v", "k_pages", "v_pages", "k_scale", "v_scale", "q", "out"])
@pytest.mark.parametrize("mode", ["reverse", "forward"])
def test_inputs_that_want_a_gradient_are_refused(which, mode, cuda_device):
    """No gradient is dropped in silence, whichever tensor it belongs to."""
    import torch.autograd.forward_ad as fwd
    dev = cuda_device
    ct = F32 if which in ("k_pages", "v_pages", "k", "v", "q", "out") else I8
    t = {n: torch.zeros(4, 2, 16, 64, dtype=ct, device=dev) for n in ("k_pages", "v_pages")}
    t |= {n: torch.ones(4, 2, 16, device=dev) for n in ("k_scale", "v_scale")}
    t |= {n: torch.zeros(2, 2, 1, 64, device=dev) for n in ("k", "v", "q", "out")}
    table, ln = i32([[0, 1], [2, 3]], dev), i32([20, 31], dev)

    def calls(t):
        kw = dict(scales=(t["k_scale"], t["v_scale"]) if ct == I8 else None)
        pages = t["k_pages"], t["v_pages"], table, ln
        write = lambda: mab.kv_cache_write(t["k"], t["v"], *pages, **kw)
        read = lambda: mab.kv_cache_read(*pages, 32, dtype=F32, **kw)
        into = lambda: mab.kv_cache_read(*pages, 1, dtype=F32, out=(t["out"], torch.zeros_like(t["q"])), **kw)
        attend = lambda: mab.decode_attention(t["q"], *pages, out=t["out"], **kw)
        return {"k": [write], "v": [write], "q": [attend], "out": [attend, into]}.get(
            which, [write, read, attend])

    for call in calls(t):
        call()  # as they are: no error
    with fwd.dual_level():
        if mode == "reverse":
            t[which] = t[which].requires_grad_()
        else:
            t[which] = fwd.make_dual(t[which], torch.ones_like(t[which]))
        for call in calls(t):
            with pytest.raises(RuntimeError, match="no gradient"):
                call()
        if mode == "reverse":
            with torch.no_grad():
                for call in calls(t):
                    call()
    mab.check_status(dev)


def test_workspaces_do_not_grow_with_the_streams(cuda_device):
    """A program that goes through many streams holds a few workspaces, and the results on
    each of them are the same."""
    dev, E, H, D, page, n = cuda_device, 2, 4, 64, 16, 3000
    g = torch.Generator(device=dev).manual_seed(56)
    k, v = (torch.randn(E, H, n, D, generator=g, device=dev, dtype=torch.float64) for _ in range(2))
    kp, _, table, _ = paged(k, BF16, page, 400, dev)
    vp = paged(v, BF16, page, 0, dev)[0]
    q = torch.randn(E, H, 1, D, generator=g, device=dev).to(BF16)
    ln = i32([n, n - 1], dev)
    want = mab.decode_attention(q, kp, vp, table, ln, check=True)
    torch.cuda.synchronize(dev)
    before = torch.cuda.memory_allocated(dev)
    streams = [torch.cuda.Stream(dev, priority=p) for _ in range(30) for p in (0, -1)]
    got = []
    for _ in range(2):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(mab.decode_attention(q, kp, vp, table, ln))
    torch.cuda.synchronize(dev)
    for x in got:
        assert torch.equal(x, want)
    del got, x
    assert len({s.cuda_stream for s in streams}) >= 50
    assert torch.cuda.memory_allocated(dev) - before <= 17 * 2 ** 23 * 1.3
    mab.check_status(dev)


def test_read_back_leaves_tokens_of_missing_pages_out_of_the_mask(cuda_device):
    """A page that is not there gives zeros that the mask does not call valid."""
    dev = cuda_device
    kp, vp = (torch.ones(4, 2, 16, 64, dtype=BF16, device=dev) for _ in range(2))
    table, ln = i32([[0, 4], [-1, 3]], dev), i32([20, 32], dev)
    k, v, mask = mab.kv_cache_read(kp, vp, table, ln, 32)
    with pytest.raises(mab.MonarchAttentionError, match="page that is not there"):
        mab.check_status(dev)
    want = torch.zeros(2, 32, dtype=torch.bool, device=dev)
    want[0, :16] = want[1, 16:] = True
    assert torch.equal(mask, want)
    for x in (k, v):
        assert torch.equal(x, want[:, None, :, None].expand_as(x).to(BF16))


def test_appending_never_waits_for_the_device(cuda_device):
    """New pages do not make the host wait."""
    dev, E, Hk, D = cuda_device, 3, 2, 64
    cache = mab.PagedKVCache(40, Hk, D, max_seqs=E, max_len=64, page_size=4, dtype=BF16, device=dev)
    g = torch.Generator(device=dev).manual_seed(57)
    xs = [torch.randn(E, Hk, 2, D, generator=g, device=dev).to(BF16) for _ in range(12)]
    q = xs[0][:, :, :1].contiguous()
    cache.append(xs[0], xs[0])  # first use of every kernel
    cache.attend(q)
    torch.cuda.synchronize(dev)
    mode = torch.cuda.get_sync_debug_mode()
    try:
        torch.cuda.set_sync_debug_mode("error")
        for x in xs[1:]:
            cache.append(x, x)
            cache.attend(q)
    finally:
        torch.cuda.set_sync_debug_mode(mode)
    mab.check_status(dev)
    assert cache.lengths.tolist() == [24] * E
    k, v, mask = cache.read()
    assert mask.all() and torch.equal(k, torch.cat(xs, 2)) and torch.equal(v, k)


def test_appending_counts_that_the_host_knows_never_waits(cuda_device):
    """Counts as a list: sequences that take nothing, or less, without a wait."""
    dev, E, Hk, D = cuda_device, 3, 2, 64
    cache = mab.PagedKVCache(40, Hk, D, max_seqs=E, max_len=64, page_size=4, dtype=I8, device=dev)
    g = torch.Generator(device=dev).manual_seed(58)
    xs = [torch.randn(E, Hk, 2, D, generator=g, device=dev).to(BF16) for _ in range(30)]
    took = [2, 0, 1]
    cache.append(xs[0], xs[0], count=took)  # first use of every kernel
    torch.cuda.synchronize(dev)
    mode = torch.cuda.get_sync_debug_mode()
    try:
        torch.cuda.set_sync_debug_mode("error")
        for x in xs[1:]:
            cache.append(x, x, count=took)
    finally:
        torch.cuda.set_sync_debug_mode(mode)
    mab.check_status(dev)
    assert cache.lengths.tolist() == [60, 0, 30] and cache.free_pages == 40 - 15 - 8
    plain = mab.PagedKVCache(40, Hk, D, max_seqs=E, max_len=64, page_size=4, dtype=I8, device=dev)
    x = torch.cat([torch.cat([x[:, :, :1] for x in xs], 2), torch.cat([x[:, :, 1:] for x in xs], 2)], 2)
    x[0] = torch.cat(xs, 2)[0]
    plain.append(x, x, count=[60, 0, 30])
    for a, b in zip(cache.read(64), plain.read(64)):
        assert torch.equal(a, b)


def test_counts_on_the_device_end_in_no_false_refusal(cuda_device):
    """Bounds that drifted from the lengths are made exact before a call is refused, and
    pages taken for nothing come back."""
    dev, E, Hk, D = cuda_device, 3, 2, 64
    cache = mab.PagedKVCache(12, Hk, D, max_seqs=E, max_len=16, page_size=2, dtype=BF16, device=dev)
    g = torch.Generator(device=dev).manual_seed(59)
    kept = [[], [], []]
    for step in range(40):
        x = torch.randn(E, Hk, 2, D, generator=g, device=dev).to(BF16)
        n = [2 if step < 4 else 0, 1 if step % 4 == 0 else 0, 0]
        cache.append(x, x, count=i32(n, dev), check=True)
        for e in range(E):
            kept[e].append(x[e, :, : n[e]])
    assert cache.lengths.tolist() == [8, 10, 0]
    cache.tighten()
    assert cache.free_pages == 12 - 4 - 5
    k, v, mask = cache.read()
    assert k.shape[2] == 10
    for e in range(E):
        want = torch.cat(kept[e], 1)
        n = want.shape[1]
        assert torch.equal(k[e, :, :n], want) and torch.equal(v[e, :, :n], want) and int(mask[e].sum()) == n
    x = torch.zeros(E, Hk, 2, D, dtype=BF16, device=dev)
    cache.append(x, x, count=i32([0, 2, 2], dev), check=True)  # one page is left
    with pytest.raises(RuntimeError, match="full"):
        cache.append(x, x, count=i32([2, 2, 0], dev))
    cache.append(x, x, count=i32([2, 0, 0], dev), check=True)
    assert cache.lengths.tolist() == [10, 12, 2] and cache.free_pages == 0
    cache.free(1)
    for _ in range(3):
        cache.append(x, x, count=i32([2, 0, 0], dev), check=True)
    with pytest.raises(ValueError, match="max_len"):
        cache.append(x, x, count=i32([1, 0, 0], dev))
    cache.append(x, x, count=i32([0, 0, 1], dev), check=True)
    assert cache.lengths.tolist() == [16, 0, 3]
