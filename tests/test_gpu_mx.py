"""Microscaled (MX) operators on a B200 against the 64-bit oracle (oracle/mx_oracle.py).

Tolerances, derived from the number formats:
  * quantisation is exact: codes and scale bytes equal the oracle's;
  * products: the elements' products and scales are exact in fp32, so a sum over K differs
    from the 64-bit one by the accumulation alone.  An instruction adds 32 products to the
    accumulator with at least 24 bits kept below the largest of them: at most
    33 * 2^-23 * S for K/32 instructions, S = sum |x w|, i.e. less than 1.04 K 2^-23 S
    (ACC below; S is computed per output);
  * bf16 outputs add half a step, 2^-9 of the value's binade: at most 2^-8 relative;
  * MX8 outputs add half an e4m3 step: 2^-4 relative, or 2^-10 of the block's scale below
    the type's normal range, and the exponential and reciprocal 2^-20 relative.
"""
from __future__ import annotations

import pytest
import torch

from easyinfra_b200 import ops
from oracle import mx_oracle as M

pytestmark = pytest.mark.gpu
bf = torch.bfloat16


def gen(device, seed):
    g = torch.Generator(device=device)
    g.manual_seed(seed)
    return g


def codes_of(q: ops.MX8Rows):
    return q.buf[:, :q.K].contiguous(), q.buf[:, q.K:q.K + q.K // 32].contiguous()


# ------------------------------------------------------------------ quantisation
def awkward(rows, K, dtype, device, seed):
    """Values over many binades, with whole blocks of zeros, of the largest and of the
    smallest magnitudes, borders of the scale and exact ties of the element grids."""
    g = gen(device, seed)
    x = torch.randn(rows, K, generator=g, device=device)
    x = x * torch.exp2(torch.randint(-30, 30, (rows, K // 32, 1), generator=g, device=device).float()).expand(
        rows, K // 32, 32).reshape(rows, K)
    b = x.view(-1, 32)
    n = b.shape[0]
    b[0] = 0
    if n > 8:
        b[1], b[2] = 0, 0
        b[1, 5] = 448.0 * 4          # the largest value exactly on both borders
        b[2, 31] = -6.0 * 2.0 ** -9
        b[3] = torch.finfo(dtype).max
        b[4] = torch.finfo(dtype).smallest_normal
        b[5] = torch.linspace(-8, 7.5, 32, device=device) / 8   # ties of e2m1 and e4m3
        b[5, 0] = 6.0
        b[6] = -0.0
        b[7] = 2.0 ** -133           # subnormal
    return x.to(dtype)


@pytest.mark.parametrize("dtype", [bf, torch.float32])
@pytest.mark.parametrize("rows,K", [(1, 32), (3, 96), (5, 160), (1, 4096), (257, 1408), (1000, 544)])
def test_quantisation_is_exact(cuda_device, rows, K, dtype):
    x = awkward(rows, K, dtype, cuda_device, rows + K)
    q8 = ops.quantize_mx8(x)
    d4, s4 = ops.quantize_mx4(x)
    v8, v4 = ops.dequantize_mx8(q8, torch.float32), ops.dequantize_mx4(d4, s4, torch.float32)
    b8, b4 = ops.dequantize_mx8(q8, bf), ops.dequantize_mx4(d4, s4, bf)
    torch.cuda.synchronize()
    c, e = M.quantize(x, False)
    got_c, got_e = codes_of(q8)
    assert torch.equal(got_e, e) and torch.equal(got_c, c)
    assert not q8.buf[:, K + K // 32:].any()                    # padding
    val = M.values(c, e, False)
    assert torch.equal(v8.double(), val.float().double()) and torch.equal(b8, val.float().to(bf))
    c, e = M.quantize(x, True)
    assert torch.equal(s4, e) and torch.equal(d4, M.pack4(c))
    val = M.values(c, e, True)
    assert torch.equal(v4.double(), val.float().double()) and torch.equal(b4, val.float().to(bf))


@pytest.mark.parametrize("dtype", [bf, torch.float32])
def test_quantisation_of_nan_and_infinity(cuda_device, dtype):
    x = torch.randn(4, 128, generator=gen(cuda_device, 0), device=cuda_device).to(dtype)
    x[0, 3], x[1, 40], x[2, 127] = float("nan"), float("inf"), float("-inf")
    q8 = ops.quantize_mx8(x)
    d4, s4 = ops.quantize_mx4(x)
    v8, v4 = ops.dequantize_mx8(q8), ops.dequantize_mx4(d4, s4)
    bad = ~torch.isfinite(x.view(4, 4, 32)).all(-1, keepdim=True).expand(4, 4, 32).reshape(4, 128)
    for v in (v8, v4):
        assert torch.equal(torch.isnan(v), bad) and torch.isfinite(v[~bad]).all()
    assert torch.equal(s4 == 255, bad.view(4, 4, 32)[..., 0])


def test_quantisation_of_strided_and_empty(cuda_device):
    d = cuda_device
    wide = torch.randn(37, 512, generator=gen(d, 1), device=d).to(bf)
    view = wide[:, 128:352]
    a, b = ops.quantize_mx8(view), ops.quantize_mx8(view.contiguous())
    assert torch.equal(a.buf, b.buf)
    for u, v in zip(ops.quantize_mx4(view), ops.quantize_mx4(view.contiguous())):
        assert torch.equal(u, v)
    rowless = wide[:1].expand(5, 512)                       # stride 0
    assert torch.equal(ops.quantize_mx8(rowless).buf[4], ops.quantize_mx8(wide[:1]).buf[0])
    w3 = torch.randn(3, 64, 96, generator=gen(d, 2), device=d)
    dd, ss = ops.quantize_mx4(w3)
    assert dd.shape == (3, 64, 48) and ss.shape == (3, 64, 3)
    assert torch.equal(dd.view(-1, 48), ops.quantize_mx4(w3.view(-1, 96))[0])
    assert ops.quantize_mx8(wide[:0]).buf.shape == (0, ops.mx8_row_bytes(512))
    assert ops.dequantize_mx4(*ops.quantize_mx4(wide[:0])).shape == (0, 512)
    big = torch.zeros(37, 1024, dtype=torch.uint8, device=d)
    big.fill_(7)
    out = ops.quantize_mx8(view, out=ops.MX8Rows(big[:, 16:16 + 240], 224))
    assert torch.equal(out.buf[:, :231], b.buf[:, :231])
    assert (big[:, :16] == 7).all() and (big[:, 256:] == 7).all()


# ------------------------------------------------------------------ prologue
@pytest.mark.parametrize("dtype", [bf, torch.float32])
@pytest.mark.parametrize("T,H", [(1, 32), (1, 2048), (7, 1408), (333, 4096), (64, 96), (2, 8192)])
@pytest.mark.parametrize("add", [True, False])
def test_add_rmsnorm_mx8(cuda_device, T, H, dtype, add):
    d = cuda_device
    g = gen(d, T * H)
    res = (3 * torch.randn(T, H, generator=g, device=d)).to(dtype)
    hid = torch.randn(T, H, generator=g, device=d).to(dtype) if add else None
    w = (1 + 0.2 * torch.randn(H, generator=g, device=d)).to(dtype)
    if T > 5:
        res[3] = 0
        if add:
            hid[3] = 0
    keep = res.clone()
    ro, nm, q = ops.add_rmsnorm_mx8(res, hid, w, 1e-6)
    r2, n2 = ops.add_rmsnorm(res, hid, w, 1e-6)
    assert torch.equal(res, keep)
    assert torch.equal(ro, r2) and torch.equal(q.buf, ops.quantize_mx8(nm).buf)
    # 1/rms is within 2^-23 of the formula's (the at most 32 squares a thread sums in fp32,
    # halved by the root, and its own rounding), the product with it another 2^-24: before
    # the first rounding a value is off by less than 2^-22, so that rounding differs by at
    # most a step, the product with the weight carries that on and rounds once more
    r3, n3 = M.add_rmsnorm(res, hid, w, 1e-6)
    assert torch.equal(ro, r3)
    eps = torch.finfo(dtype).eps
    for other in (n3, n2):
        assert ((nm.double() - other.double()).abs() <= (2 * eps + 2.0 ** -21) * other.double().abs() + 1e-30).all()
    if dtype == bf:  # and that happens only next to a border: 2^-22 of a value in a step of 2^-8
        assert (nm != n3).double().mean() <= 1e-3
    _, none, q3 = ops.add_rmsnorm_mx8(res, hid, w, 1e-6, norm=False)
    assert none is None and torch.equal(q3.buf, q.buf)
    ro4, _, q4 = ops.add_rmsnorm_mx8(res, hid, w, 1e-6, residual_out=res)      # in place
    assert ro4 is res and torch.equal(res, ro) and torch.equal(q4.buf, q.buf)


def test_add_rmsnorm_mx8_strides_and_refusals(cuda_device):
    d = cuda_device
    wide = torch.randn(9, 512, generator=gen(d, 5), device=d).to(bf)
    hid = torch.randn(9, 256, generator=gen(d, 6), device=d).to(bf)
    w = torch.ones(256, device=d, dtype=bf)
    view = wide[:, 128:384]
    base = ops.add_rmsnorm_mx8(view.contiguous(), hid, w)
    for h in (hid, torch.cat([hid, hid], 1)[:, :256]):
        got = ops.add_rmsnorm_mx8(view, h, w)
        assert all(torch.equal(a, b) for a, b in zip(got[:2], base[:2])) and torch.equal(got[2].buf, base[2].buf)
    assert ops.add_rmsnorm_mx8(view[:0], None, w)[2].rows == 0
    x = hid.clone()
    for bad, kind in ((lambda: ops.add_rmsnorm_mx8(x, hid[:4], w), ValueError),
                      (lambda: ops.add_rmsnorm_mx8(x, hid, w.float()), ValueError),
                      (lambda: ops.add_rmsnorm_mx8(x[:, :40].contiguous(), None, w[:40]), ValueError),
                      (lambda: ops.add_rmsnorm_mx8(x.half(), None, w.half()), TypeError),
                      (lambda: ops.add_rmsnorm_mx8(x[:8], None, w, residual_out=x[1:]), ValueError),
                      (lambda: ops.add_rmsnorm_mx8(x, None, w, out=ops.quantize_mx8(x[:3])), ValueError)):
        with pytest.raises(kind):
            bad()


# ------------------------------------------------------------------ products
def problem(device, counts, N, K, seed, first=0, extra=0):
    """MX8 rows, offsets, MX4 weights, and their values in 64 bits."""
    g = gen(device, seed)
    P, rows = len(counts), first + sum(counts) + extra
    x = torch.randn(rows, K, generator=g, device=device)
    x = x * torch.exp2(torch.randint(-3, 4, (rows, K // 32), generator=g, device=device).float()).repeat_interleave(32, 1)
    q = ops.quantize_mx8(x)
    d, s = ops.quantize_mx4(0.05 * torch.randn(P, N, K, generator=g, device=device)
                            * torch.exp2(torch.randint(-2, 3, (P, N, 1), generator=g, device=device).float()))
    offs = [first]
    for c in counts:
        offs.append(offs[-1] + c)
    xv = M.values(*codes_of(q), False)
    wv = M.values(M.unpack4(d), s, True)
    return q, torch.tensor(offs, dtype=torch.int32, device=device), d, s, xv, wv


CASES = [  # counts, H, I
    ([1], 128, 128),
    ([3, 0, 1, 32, 0], 256, 128),                 # decode tiles, empty experts
    ([0, 0, 0], 128, 128),
    ([33, 64, 65, 1], 384, 256),                  # tiles that end inside, H % 256 != 0
    ([129, 0, 300, 128], 256, 384),
    ([1] * 40, 2048, 768),
    ([500, 31], 512, 1408),                       # 11 k-blocks: the last group of scales is ragged
    ([1000], 640, 640),
]


# rows per expert that the hint promises -> kernel: weight streaming, single-CTA tiles, CTA
# pairs (where the weight rows are a multiple of 256; tiles elsewhere)
HINTS = {"stream": 1, "tiles": 100, "pairs": 10000}


@pytest.mark.parametrize("max_ctas", [None, "4"])
@pytest.mark.parametrize("kernel", sorted(HINTS))
@pytest.mark.parametrize("counts,H,I", CASES)
def test_products(cuda_device, monkeypatch, counts, H, I, kernel, max_ctas):
    if max_ctas:  # many tiles per CTA
        monkeypatch.setenv("B200MOE_GEMM_MAX_CTAS", max_ctas)
    check_products(cuda_device, counts, H, I, rows_hint=HINTS[kernel] * len(counts))


@pytest.mark.parametrize("counts,H,I", [([1000, 700], 512, 1408), ([56] * 3, 128, 128), ([57] * 3, 256, 128),
                                        ([1] * 7, 4096, 256), ([65, 64, 1], 128, 2048)])
def test_products_without_a_hint(cuda_device, counts, H, I):
    check_products(cuda_device, counts, H, I)


def check_products(d, counts, H, I, first=0, extra=0, **kw):
    P, rows, end = len(counts), first + sum(counts) + extra, first + sum(counts)
    status = torch.zeros(1, dtype=torch.int32, device=d)
    # down
    q, offs, wd, ws, xv, wv = problem(d, counts, H, I, 1 + H + I, first, extra)
    out = torch.full((rows, H), 7.0, dtype=bf, device=d)
    y = ops.grouped_down_mx4(q, offs, ops.pack_mx4_weights(wd, ws, swiglu=False), out=out, status=status, **kw)
    ref, tot = M.grouped(xv, offs, wv), M.grouped(xv.abs(), offs, wv.abs())
    err = (y.double() - ref).abs()[first:end]
    tol = (2.0 ** -8 * ref.abs() + 1.04 * I * 2.0 ** -23 * tot)[first:end]
    assert y is out and (err <= tol).all(), float((err / tol.clamp_min(1e-30)).max())
    assert (y[:first] == 7).all() and (y[end:] == 7).all()
    # swiglu
    q, offs, wd, ws, xv, wv = problem(d, counts, 2 * I, H, 2 + H + I, first, extra)
    buf = torch.full((rows, ops.mx8_row_bytes(I)), 9, dtype=torch.uint8, device=d)
    act = ops.grouped_swiglu_mx4(q, offs, ops.pack_mx4_weights(wd, ws, swiglu=True), out=ops.MX8Rows(buf, I),
                                 status=status, **kw)
    torch.cuda.synchronize()
    assert int(status.item()) == 0
    gu, tot = M.grouped(xv, offs, wv), M.grouped(xv.abs(), offs, wv.abs())
    check_act(act, gu, tot, H, first, end)
    keep = buf.clone()
    keep[first:end, :I + I // 32] = 9
    assert (keep == 9).all()                       # rows outside and the padding are left


def check_act(act, gu, tot, H, first, end):
    """MX8 activations against silu(g) * u in 64 bits."""
    I = act.K
    codes, byte = codes_of(act)
    got = M.values(codes, byte, False)[first:end]
    ref = M.swiglu(gu)[first:end]
    if ref.numel() == 0:
        return
    g, u = gu.chunk(2, -1)
    dg, du = (1.04 * H * 2.0 ** -23 * t for t in tot.chunk(2, -1))
    acc = (1.1 * dg * u.abs() + (g / (1 + torch.exp(-g))).abs() * du + 1.1 * dg * du)[first:end] + 2.0 ** -20 * ref.abs()
    _, want = M.quantize(ref, False)
    have = byte[first:end]
    amax = ref.abs().unflatten(-1, (-1, 32)).amax(-1)
    slack = acc.unflatten(-1, (-1, 32)).amax(-1)
    # a scale differs only where the block's largest value is that near to its border
    border = 448.0 * M.scale_values(torch.minimum(want, have))
    off = want != have
    assert ((amax - border).abs()[off] <= slack[off]).all()
    assert ((want.int() - have.int()).abs() <= 1).all()
    scale = M.scale_values(torch.maximum(want, have)).repeat_interleave(32, 1)
    tol = 2.0 ** -4 * (ref.abs() + acc) + 2.0 ** -10 * scale + acc
    err = (got - ref).abs()
    assert (err <= tol).all(), float((err / tol).max())


def test_products_leave_other_rows(cuda_device):
    """Rows before the first segment and behind the last one are left as they were, with
    more allocated rows than routed ones."""
    for hint in HINTS.values():
        check_products(cuda_device, [5, 0, 70], 256, 128, first=3, extra=200, rows_hint=3 * hint)
        check_products(cuda_device, [130, 2, 0, 257], 512, 128, first=1, extra=7, rows_hint=4 * hint)


@pytest.mark.parametrize("kernel", sorted(HINTS))
def test_row_map_and_bad_tables(cuda_device, kernel):
    d = cuda_device
    counts, H, I = [20, 0, 13], 256, 128
    q, offs, wd, ws, xv, wv = problem(d, counts, H, I, 11)
    w = ops.pack_mx4_weights(wd, ws, swiglu=False)
    hint = HINTS[kernel] * 3
    down = lambda *a, **k: ops.grouped_down_mx4(*a, rows_hint=hint, **k)  # noqa: E731
    base = down(q, offs, w)
    perm = torch.randperm(40, generator=gen(d, 1), device=d)[:33].to(torch.int32)
    out = torch.full((40, H), 5.0, dtype=bf, device=d)
    down(q, offs, w, out=out, out_row_map=perm)
    assert torch.equal(out[perm.long()], base)
    rest = torch.ones(40, dtype=torch.bool, device=d)
    rest[perm.long()] = False
    assert (out[rest] == 5).all()
    # entries outside out are skipped and recorded
    status = torch.zeros(1, dtype=torch.int32, device=d)
    bad = perm.clone()
    bad[4], bad[30] = 40, -1
    out2 = torch.full((40, H), 5.0, dtype=bf, device=d)
    down(q, offs, w, out=out2, out_row_map=bad, status=status)
    assert int(status.item()) == 3
    good = torch.tensor([i for i in range(33) if i not in (4, 30)], device=d)
    assert torch.equal(out2[perm[good].long()], base[good])
    assert (out2[perm[4].long()] == 5).all() and (out2[perm[30].long()] == 5).all()
    # offsets outside the rows or descending are clamped and recorded
    for table in ([0, 20, 20, 1000], [-5, 20, 10, 33], [0, 50, 20, 33]):
        status.zero_()
        y = down(q, torch.tensor(table, dtype=torch.int32, device=d), w, status=status)
        torch.cuda.synchronize()
        assert int(status.item()) == 3 and torch.equal(y[:20], base[:20])


@pytest.mark.parametrize("kernel", sorted(HINTS))
def test_nan_reaches_its_row_alone(cuda_device, kernel):
    d, hint = cuda_device, 2 * HINTS[kernel]
    x = torch.randn(40, 256, generator=gen(d, 3), device=d)
    x[7, 100], x[33, 3] = float("nan"), float("inf")
    q = ops.quantize_mx8(x)
    wd, ws = ops.quantize_mx4(0.05 * torch.randn(2, 256, 256, generator=gen(d, 4), device=d))
    offs = torch.tensor([0, 35, 40], dtype=torch.int32, device=d)
    y = ops.grouped_down_mx4(q, offs, ops.pack_mx4_weights(wd, ws, swiglu=False), rows_hint=hint)
    act = ops.grouped_swiglu_mx4(q, offs, ops.pack_mx4_weights(wd, ws, swiglu=True), rows_hint=hint)
    nan = torch.zeros(40, dtype=torch.bool, device=d)
    nan[[7, 33]] = True
    for v in (y, ops.dequantize_mx8(act)):
        assert torch.isnan(v[nan]).all() and torch.isfinite(v[~nan]).all()


def test_product_refusals(cuda_device):
    d = cuda_device
    q, offs, wd, ws, _, _ = problem(d, [4, 4], 256, 128, 1)
    down, gu = ops.pack_mx4_weights(wd, ws, swiglu=False), ops.pack_mx4_weights(wd, ws, swiglu=True)
    for bad, kind in ((lambda: ops.grouped_down_mx4(q, offs, gu), ValueError),
                      (lambda: ops.grouped_swiglu_mx4(q, offs, down), ValueError),
                      (lambda: ops.grouped_down_mx4(q, offs[:2], down), ValueError),
                      (lambda: ops.grouped_down_mx4(q, offs, down, out=torch.empty(7, 256, dtype=bf, device=d)), ValueError),
                      (lambda: ops.grouped_down_mx4(q, offs, down, out=torch.empty(8, 256, device=d)), ValueError),
                      (lambda: ops.grouped_down_mx4(q, offs, down, out_row_map=offs), ValueError),
                      (lambda: ops.grouped_down_mx4(q.buf, offs, down), TypeError),
                      (lambda: ops.grouped_down_mx4(ops.MX8Rows(q.buf, 256), offs, down), ValueError)):
        with pytest.raises(kind):
            bad()
    wd, ws = ops.quantize_mx4(torch.zeros(513, 128, 128, device=d, dtype=bf))
    with pytest.raises(Exception, match="slot limit"):
        ops.grouped_down_mx4(q, torch.zeros(514, dtype=torch.int32, device=d), ops.pack_mx4_weights(wd, ws, swiglu=False))
    empty = ops.MX8Rows(q.buf[:0], 128)
    assert ops.grouped_down_mx4(empty, torch.zeros_like(offs), down).shape == (0, 256)
