"""The MLP layer's operators: gemm_linear, gemm_linear_dx, gemm_linear_dw, gemm_act_grad, gemm_dropout.

Results are compared with the formulas in 64 bits.  Tolerances are bounds, counted from the roundings:

  product   a sum of K products of 16-bit values in f32 by the tensor cores, which cut rather than round when
            they add: at most one unit in the last place of the partial sums' bound S = sum |a||b| for each of
            the K/16 steps and 16 more inside one, so S (K/16 + 16) 2^-23
  act       exp and the division err by a few units (exp's bound is 2 + 1.2 |t| of them), which s (1 - s) damps
            in a sigmoid: |z| 2^-20 covers forward and slope; errors of z pass with a factor of at most 1.2
  result    half a step of the result's type (eps / 2 relative), and half the smallest subnormal
"""
import ctypes
import math

import numpy as np
import pytest

from mlpgemm import lib as G

ACT_NAMES = list(G.ACTS)
torch = None


@pytest.fixture(autouse=True)
def _torch(request):
    global torch
    if request.node.get_closest_marker("gpu"):
        import torch as t
        torch = t


# ---- the generator ------------------------------------------------------------------------
def philox(ctr, key):
    """Philox4x32-10 on Python integers."""
    c, k = list(ctr), list(key)
    for _ in range(10):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [(b >> 32) ^ c[1] ^ k[0], b & 0xFFFFFFFF, (a >> 32) ^ c[3] ^ k[1], a & 0xFFFFFFFF]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return c


def test_philox_known_answers():
    # the published vectors of Philox4x32-10
    assert philox([0] * 4, [0] * 2) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    assert philox([0xFFFFFFFF] * 4, [0xFFFFFFFF] * 2) == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]
    assert philox([0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344], [0xA4093822, 0x299F31D0]) == \
        [0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1]


def factors(rows, cols, p, seed, offset, first=0):
    """Dropout's factor of every element of rows first .. first + rows - 1, in 64 bits, from the generator in numpy."""
    t = int(np.rint(p * 65536))
    groups = (cols + 7) // 8
    u = np.uint64
    c = [np.broadcast_to(np.arange(groups, dtype=u), (rows, groups)),
         np.broadcast_to(np.arange(first, first + rows, dtype=u)[:, None], (rows, groups)),
         np.full((rows, groups), offset & 0xFFFFFFFF, u), np.full((rows, groups), (offset >> 32) & 0xFFFFFFFF, u)]
    k = [seed & 0xFFFFFFFF, seed >> 32]
    m, s = u(0xFFFFFFFF), u(32)
    for _ in range(10):
        a, b = c[0] * u(0xD2511F53), c[2] * u(0xCD9E8D57)
        c = [(b >> s) ^ c[1] ^ u(k[0]), b & m, (a >> s) ^ c[3] ^ u(k[1]), a & m]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    bits = np.stack([(c[i // 2] >> u(16 * (i % 2))) & u(0xFFFF) for i in range(8)], -1).reshape(rows, -1)[:, :cols]
    return np.where(bits >= t, 65536.0 / (65536 - t) if t < 65536 else 0.0, 0.0)


def test_factors_follow_the_generator():
    seed, offset = 0x0123456789ABCDEF, 0xFEDCBA9876543210
    f = factors(3, 20, 0.25, seed, offset)
    w = philox([1, 2, offset & 0xFFFFFFFF, offset >> 32], [seed & 0xFFFFFFFF, seed >> 32])   # row 2, columns 8..15
    half = [(w[i // 2] >> (16 * (i % 2))) & 0xFFFF for i in range(8)]
    assert [x != 0 for x in f[2, 8:16]] == [h >= 16384 for h in half]
    assert set(np.unique(f)) == {0.0, 65536 / 49152}
    big = factors(256, 512, 0.1, 1, 2)
    n, q = big.size, 6554 / 65536
    assert abs((big == 0).mean() - q) < 5 * math.sqrt(q * (1 - q) / n)     # five standard deviations


# ---- formulas in 64 bits --------------------------------------------------------------------
def act64(z, act):
    if act == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if act == "gelu":
        return 0.5 * z * torch.special.erfc(-z / 2 ** 0.5)
    if act == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh((2 / math.pi) ** 0.5 * (z + 0.044715 * z ** 3)))
    if act == "silu":
        return z * torch.sigmoid(z)
    return z


def slope64(z, act):
    """The derivative by central differences of the function above, in 64 bits (error about 1e-10)."""
    if act == "none":
        return torch.ones_like(z)
    if act == "relu":
        return (z > 0).double()
    h = 1e-5
    return (act64(z + h, act) - act64(z - h, act)) / (2 * h)


def ttype(name):
    return {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}[name]


def half_step(ref, dtype):
    fi = torch.finfo(dtype)
    return ref.abs() * (fi.eps / 2) + fi.smallest_normal * fi.eps / 2


def rand(shape, dtype, seed, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda", dtype=torch.float32) * scale).to(dtype)


def strided(shape, dtype, ld, shift=0, fill=None):
    """A [rows, cols] view with `ld` elements between rows, `shift` elements into its buffer."""
    rows, cols = shape
    buf = torch.empty(shift + rows * ld, dtype=dtype, device="cuda")
    if fill is not None:
        buf.fill_(fill)
    return buf, buf[shift:].as_strided((rows, cols), (ld, 1))


def put(x, ld, shift=0):
    """A copy of x with `ld` elements between rows, NaN between them."""
    _, v = strided(x.shape, x.dtype, ld, shift, float("nan"))
    v.copy_(x)
    return v


def workspace(op, A, B, N, K, M, lda=0, ldb=0):
    n = G.linear_workspace(op, A, B, N, K, M, lda, ldb)
    return (torch.empty(n, dtype=torch.uint8, device="cuda"), n) if n else (None, 0)


def stream():
    return torch.cuda.current_stream().cuda_stream


def assert_close(out, ref, tol, what):
    out = out.double()
    assert torch.equal(torch.isnan(out), torch.isnan(ref)), what + ": NaN in other places"
    inf = torch.isinf(ref)
    assert torch.equal(out[inf], ref[inf]), what
    ok = torch.isfinite(ref)
    over = (out - ref).abs()[ok] - (tol.expand_as(ref)[ok])
    assert over.numel() == 0 or float(over.max()) <= 0, f"{what}: {float(over.max()):.3g} past its bound"


def product_error(a, b, depth):
    """The bound on a product's error before its epilogue."""
    return (a.double().abs() @ b.double().abs()) * ((depth / 16 + 16) * 2.0 ** -23)


def linear_ref(x, w, bias, res, act, p, seed, offset):
    """(Y, Z) in 64 bits and the bounds on their errors."""
    t = x.dtype
    z = x.double() @ w.double()
    e = product_error(x, w, x.shape[1])
    if bias is not None:
        z = z + bias.double()
    ez = e + z.abs() * 2.0 ** -23
    y = act64(z, act)
    ey = ez * 1.2 + (0 if act == "none" else z.abs() * 2.0 ** -20)
    if p:
        f = torch.from_numpy(factors(*y.shape, p, seed, offset)).cuda()
        y = torch.where(f == 0, torch.zeros_like(y), y * f)
        ey = torch.where(f == 0, torch.zeros_like(y), ey * f + y.abs() * 2.0 ** -23)
    if res is not None:
        y = res.double() + y
        ey = ey + y.abs() * 2.0 ** -23
    return y, z, ey + half_step(y, t) * 1.01, ez + half_step(z, t) * 1.01


SIZES = [(1, 1, 1), (1, 64, 8), (2, 4096, 264), (3, 7, 5), (13, 520, 1000), (16, 129, 24), (17, 100, 33),
         (40, 64, 136), (65, 72, 257), (128, 512, 256), (130, 257, 264), (200, 1000, 520), (257, 640, 1032),
         (700, 96, 2056), (1100, 520, 1288), (1300, 136, 2056), (1030, 77, 2571), (2310, 1160, 1112), (4200, 64, 808), (3, 264, 10000), (31, 1090, 10112),
         (16, 192, 11008), (9, 4104, 4096), (201, 40, 10023), (2200, 646, 40), (1124, 67, 43), (536, 66, 41),
         (320, 144, 37)]


@pytest.mark.gpu
@pytest.mark.parametrize("type", ["f16", "bf16"])
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_linear_sizes(gemm, size, type):
    N, K, M = size
    t = ttype(type)
    x, w = rand((N, K), t, 1), rand((K, M), t, 2, K ** -0.5)
    b, r = rand((M,), t, 3), rand((N, M), t, 4)
    y, z = torch.empty(N, M, dtype=t, device="cuda"), torch.empty(N, M, dtype=t, device="cuda")
    ws, wsb = workspace(G.OP_LINEAR, x, w, N, K, M)
    G.linear(0, G.TYPES[type], x, w, y, N, K, M, bias=b, act=G.ACTS["silu"], residual=r, preact=z, dropout_p=0.3,
             seed=77, offset=1 << 40, workspace=ws, workspace_bytes=wsb, stream=stream())
    G.sync(0, stream())
    ry, rz, ty, tz = linear_ref(x, w, b, r, "silu", 0.3, 77, 1 << 40)
    assert_close(z, rz, tz, "Z")
    assert_close(y, ry, ty, "Y")
    y2 = torch.full_like(y, float("nan"))
    G.linear(0, G.TYPES[type], x, w, y2, N, K, M, workspace=ws, workspace_bytes=wsb, stream=stream())
    G.sync(0, stream())
    ry, _, ty, _ = linear_ref(x, w, None, None, "none", 0, 0, 0)
    assert_close(y2, ry, ty, "the bare product")


@pytest.mark.gpu
@pytest.mark.parametrize("act", ACT_NAMES)
@pytest.mark.parametrize("N,M", [(5, 328), (300, 328), (1300, 2056)])
@pytest.mark.parametrize("bias,res,pre,p", [(1, 0, 0, 0.0), (0, 1, 0, 0.0), (0, 0, 1, 0.0), (0, 0, 0, 0.5),
                                            (0, 1, 1, 1.0), (1, 1, 1, 0.1)])
def test_linear_epilogues(gemm, act, N, M, bias, res, pre, p):
    K, t = 200, torch.bfloat16
    x, w = rand((N, K), t, 1, 2.0), rand((K, M), t, 2, K ** -0.5)
    b = rand((M,), t, 3) if bias else None
    r = rand((N, M), t, 4) if res else None
    y = torch.empty(N, M, dtype=t, device="cuda")
    z = torch.empty(N, M, dtype=t, device="cuda") if pre else None
    G.linear(0, G.TYPES["bf16"], x, w, y, N, K, M, bias=b, act=G.ACTS[act], residual=r, preact=z, dropout_p=p,
             seed=2 ** 64 - 3, offset=5, stream=stream())
    G.sync(0, stream())
    ry, rz, ty, tz = linear_ref(x, w, b, r, act, p, 2 ** 64 - 3, 5)
    assert_close(y, ry, ty, "Y")
    if pre:
        assert_close(z, rz, tz, "Z")
    if p == 1.0:
        assert torch.equal(y, r)


@pytest.mark.gpu
@pytest.mark.parametrize("N,M", [(1, 200), (13, 200), (140, 200), (600, 200), (1290, 2000)])
@pytest.mark.parametrize("pad,shift", [(8, 8), (3, 1), (0, 1)])
def test_linear_strides_and_alignment(gemm, N, M, pad, shift):
    # rows further apart than their length, buffers that start anywhere; the gaps keep what they held
    K, t = 136, torch.float16
    x0, w0, b, r0 = rand((N, K), t, 1), rand((K, M), t, 2, K ** -0.5), rand((M,), t, 3), rand((N, M), t, 4)
    x, w, r = put(x0, K + pad, shift), put(w0, M + pad, shift), put(r0, M + pad, shift)
    b1 = torch.cat([b[:1], b])[1:]                      # two bytes past an aligned address
    ybuf, y = strided((N, M), t, M + pad, shift, 7.0)
    zbuf, z = strided((N, M), t, M + pad, shift, 7.0)
    ws, wsb = workspace(G.OP_LINEAR, x, w, N, K, M, K + pad, M + pad)
    assert (wsb == 0) == (shift == 8)
    G.linear(0, G.TYPES["f16"], x, w, y, N, K, M, bias=b1, act=G.ACTS["gelu"], residual=r, preact=z, dropout_p=0.2,
             seed=9, offset=1, ldx=K + pad, ldw=M + pad, ldy=M + pad, ldr=M + pad, ldz=M + pad, workspace=ws,
             workspace_bytes=wsb, stream=stream())
    G.sync(0, stream())
    ry, rz, ty, tz = linear_ref(x0, w0, b, r0, "gelu", 0.2, 9, 1)
    assert_close(y, ry, ty, "Y")
    assert_close(z, rz, tz, "Z")
    for buf, v in ((ybuf, y), (zbuf, z)):
        v.fill_(7.0)
        assert bool((buf == 7.0).all()), "an element between rows was written"


@pytest.mark.gpu
@pytest.mark.parametrize("N", [1, 21, 1290])
def test_odd_rows_on_aligned_pitches(gemm, N):
    # rows of odd length that start on 16 bytes: read and written in place, up to their last element and no further
    K, M, ldk, ldm, t = 133, 2003, 136, 2008, torch.bfloat16
    x0, w0, r0, dz0 = rand((N, K), t, 1), rand((K, M), t, 2, K ** -0.5), rand((N, M), t, 3), rand((N, M), t, 4)
    x, w, r, dz = put(x0, ldk), put(w0, ldm), put(r0, ldm), put(dz0, ldm)
    assert workspace(G.OP_LINEAR, x, w, N, K, M, ldk, ldm)[1] == 0
    ybuf, y = strided((N, M), t, ldm, 0, 7.0)
    zbuf, z = strided((N, M), t, ldm, 0, 7.0)
    G.linear(0, 1, x, w, y, N, K, M, act=G.ACTS["silu"], residual=r, preact=z, dropout_p=0.2, seed=9, offset=1,
             ldx=ldk, ldw=ldm, ldy=ldm, ldr=ldm, ldz=ldm, stream=stream())
    xbuf, dx = strided((N, K), t, ldk, 0, 7.0)
    G.linear_dx(0, 1, dz, w, dx, N, K, M, lddz=ldm, ldw=ldm, lddx=ldk, stream=stream())
    wbufs = []
    for out in ("bf16", "f32"):
        wbufs.append(strided((K, M), ttype(out), ldm, 0, 7.0))
        G.linear_dw(0, 1, x, dz, wbufs[-1][1], N, K, M, out_type=G.TYPES[out], ldx=ldk, lddz=ldm, lddw=ldm,
                    stream=stream())
    G.sync(0, stream())
    ry, rz, ty, tz = linear_ref(x0, w0, None, r0, "silu", 0.2, 9, 1)
    assert_close(y, ry, ty, "Y")
    assert_close(z, rz, tz, "Z")
    v = dz0.double() @ w0.double().t()
    assert_close(dx, v, product_error(dz0, w0.t(), M) + half_step(v, t) * 1.01, "dX")
    v = x0.double().t() @ dz0.double()
    for _, dw in wbufs:
        assert_close(dw, v, product_error(x0.t(), dz0, N) + half_step(v, dw.dtype) * 1.01, "dW")
    for buf, view in [(ybuf, y), (zbuf, z), (xbuf, dx)] + wbufs:
        view.fill_(7.0)
        assert bool((buf == 7.0).all()), "an element between rows was written"


@pytest.mark.gpu
@pytest.mark.parametrize("N,M", [(4, 272), (333, 272), (1300, 2056)])
def test_linear_residual_in_place(gemm, N, M):
    K, t = 264, torch.bfloat16
    x, w, r = rand((N, K), t, 1), rand((K, M), t, 2, K ** -0.5), rand((N, M), t, 4)
    y = r.clone()
    G.linear(0, G.TYPES["bf16"], x, w, y, N, K, M, residual=y, stream=stream())
    G.sync(0, stream())
    ry, _, ty, _ = linear_ref(x, w, None, r, "none", 0, 0, 0)
    assert_close(y, ry, ty, "Y")


@pytest.mark.gpu
@pytest.mark.parametrize("N,M", [(7, 264), (260, 264), (1300, 2056)])
def test_linear_specials_stay_in_their_rows(gemm, N, M):
    # an infinity or NaN in X reaches its own row alone; a dropped element is 0 whatever it held
    K, t = 72, torch.float16
    x, w = rand((N, K), t, 1), rand((K, M), t, 2, K ** -0.5)
    x[2, 3], x[4, 0] = float("nan"), float("inf")
    y = torch.empty(N, M, dtype=t, device="cuda")
    G.linear(0, G.TYPES["f16"], x, w, y, N, K, M, act=G.ACTS["relu"], dropout_p=0.5, seed=3, offset=4, stream=stream())
    G.sync(0, stream())
    f = torch.from_numpy(factors(N, M, 0.5, 3, 4)).cuda()
    assert bool(torch.isnan(y[2][f[2] != 0]).all())
    assert bool((y[f == 0] == 0).all())
    sign = w[0].double().sign()
    assert bool(torch.isinf(y[4][(f[4] != 0) & (sign > 0)]).all())
    assert bool((y[4][(f[4] != 0) & (sign < 0)] == 0).all())
    rest = [i for i in range(N) if i not in (2, 4)]
    assert bool(torch.isfinite(y[rest]).all())


GRAD_SIZES = [(1, 1, 1), (1, 264, 136), (5, 9, 7), (16, 520, 1032), (33, 257, 129), (64, 128, 128), (130, 1000, 264),
              (333, 136, 2056), (600, 520, 520), (1050, 72, 200), (2100, 256, 264), (1300, 2056, 1288), (1029, 2571, 1101), (520, 2312, 1544), (65, 2600, 2056), (5, 10240, 328), (32, 11008, 200),
              (200, 10012, 36), (2126, 34, 616), (1075, 43, 65), (1, 200, 9657), (646, 2259, 32), (68, 1119, 37),
              (1, 1073, 33), (259, 34, 136)]


@pytest.mark.gpu
@pytest.mark.parametrize("type", ["f16", "bf16"])
@pytest.mark.parametrize("size", GRAD_SIZES, ids=str)
def test_gradient_products(gemm, size, type):
    N, K, M = size
    t = ttype(type)
    x, w, dz = rand((N, K), t, 1), rand((K, M), t, 2, M ** -0.5), rand((N, M), t, 3)
    ws, wsb = workspace(G.OP_DX, dz, w, N, K, M)
    e, ref = product_error(dz, w.t(), M), dz.double() @ w.double().t()
    for res in (None, rand((N, K), t, 4)):
        dx = torch.full((N, K), float("nan"), dtype=t, device="cuda")
        G.linear_dx(0, G.TYPES[type], dz, w, dx, N, K, M, residual=res, workspace=ws, workspace_bytes=wsb,
                    stream=stream())
        G.sync(0, stream())
        v = ref if res is None else ref + res.double()
        assert_close(dx, v, e + v.abs() * 2.0 ** -23 + half_step(v, t) * 1.01, "dX")
    ws, wsb = workspace(G.OP_DW, x, dz, N, K, M)
    e, ref = product_error(x.t(), dz, N), x.double().t() @ dz.double()
    for out in (type, "f32"):
        o = ttype(out)
        for res in (None, rand((K, M), o, 5, N ** 0.5)):
            dw = torch.full((K, M), float("nan"), dtype=o, device="cuda") if res is None else res.clone()
            G.linear_dw(0, G.TYPES[type], x, dz, dw, N, K, M, out_type=G.TYPES[out],
                        residual=None if res is None else dw, workspace=ws, workspace_bytes=wsb, stream=stream())
            G.sync(0, stream())
            v = ref if res is None else ref + res.double()
            assert_close(dw, v, e + v.abs() * 2.0 ** -23 + half_step(v, o) * 1.01, f"dW in {out}")


@pytest.mark.gpu
@pytest.mark.parametrize("size", [(13, 136, 200), (300, 200, 136), (1300, 2056, 1800)], ids=str)
@pytest.mark.parametrize("pad,shift", [(8, 8), (3, 1)])
def test_gradient_products_strided(gemm, size, pad, shift):
    (N, K, M), t = size, torch.bfloat16
    x0, w0, dz0 = rand((N, K), t, 1), rand((K, M), t, 2, M ** -0.5), rand((N, M), t, 3)
    x, w, dz = put(x0, K + pad, shift), put(w0, M + pad, shift), put(dz0, M + pad, shift)
    buf, dx = strided((N, K), t, K + pad, shift, 7.0)
    ws, wsb = workspace(G.OP_DX, dz, w, N, K, M, M + pad, M + pad)
    G.linear_dx(0, G.TYPES["bf16"], dz, w, dx, N, K, M, lddz=M + pad, ldw=M + pad, lddx=K + pad, workspace=ws,
                workspace_bytes=wsb, stream=stream())
    G.sync(0, stream())
    v = dz0.double() @ w0.double().t()
    assert_close(dx, v, product_error(dz0, w0.t(), M) + half_step(v, t) * 1.01, "dX")
    dx.fill_(7.0)
    assert bool((buf == 7.0).all())
    ws, wsb = workspace(G.OP_DW, x, dz, N, K, M, K + pad, M + pad)
    for out in ("bf16", "f32"):
        o = ttype(out)
        r0 = rand((K, M), o, 6)
        r = put(r0, M + pad, shift)
        buf, dw = strided((K, M), o, M + pad, shift, 7.0)
        G.linear_dw(0, G.TYPES["bf16"], x, dz, dw, N, K, M, out_type=G.TYPES[out], residual=r, ldx=K + pad,
                    lddz=M + pad, lddw=M + pad, ldr=M + pad, workspace=ws, workspace_bytes=wsb, stream=stream())
        G.sync(0, stream())
        v = x0.double().t() @ dz0.double() + r0.double()
        assert_close(dw, v, product_error(x0.t(), dz0, N) + v.abs() * 2.0 ** -23 + half_step(v, o) * 1.01, "dW")
        dw.fill_(7.0)
        assert bool((buf == 7.0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("size,pad", [((333, 1032, 2056), 0), ((70, 2056, 1804), 8), ((600, 2100, 2058), 6),
                                      ((1, 4096, 520), 0), ((1100, 3000, 1300), 4), ((65, 1, 9000), 0)], ids=str)
def test_dw_in_place_equals_dw_beside(gemm, size, pad):
    # one addition of the same two numbers, rounded to nearest, wherever the old value comes from: the same bits
    N, K, M = size
    x, dz, r = rand((N, K), torch.bfloat16, 1), rand((N, M), torch.bfloat16, 2), rand((K, M), torch.float32, 3)
    r[0, 5], r[K // 2, 7], r[K - 1, M - 1] = float("inf"), float("nan"), 3e38
    buf, dw = strided((K, M), torch.float32, M + pad, 0, 7.0)
    dw.copy_(r)
    beside = torch.empty_like(r)
    ws, wsb = workspace(G.OP_DW, x, dz, N, K, M)
    kw = dict(out_type=G.TYPES["f32"], workspace=ws, workspace_bytes=wsb, stream=stream())
    G.linear_dw(0, G.TYPES["bf16"], x, dz, beside, N, K, M, residual=r, **kw)
    G.linear_dw(0, G.TYPES["bf16"], x, dz, dw, N, K, M, residual=dw, lddw=M + pad, ldr=M + pad, **kw)
    G.sync(0, stream())
    assert bool(torch.equal(dw.isnan(), beside.isnan()))
    assert bool(torch.equal(dw.nan_to_num(nan=0.0), beside.nan_to_num(nan=0.0)))
    dw.fill_(7.0)
    assert bool((buf == 7.0).all()), "an element between rows was written"


@pytest.mark.gpu
def test_dw_long_sum_in_32_bits(gemm):
    # accumulated over many rows, the f32 gradient stays within 1e-6 of the 64-bit sum (2-norm): partial sums of
    # 512 rows leave the tensor cores, whose adds cut, before 512/16 of them have lost 32 * 2^-25 = 1e-6
    for N, K, M in ((700, 264, 512), (4000, 264, 512), (8192, 264, 512), (16384, 64, 136), (30000, 264, 512),
                    (3000, 1032, 520), (2000, 2056, 4104), (9000, 2056, 72)):
        x, dz = rand((N, K), torch.bfloat16, 1), rand((N, M), torch.bfloat16, 2)
        dw = torch.empty(K, M, device="cuda")
        G.linear_dw(0, G.TYPES["bf16"], x, dz, dw, N, K, M, out_type=G.TYPES["f32"], stream=stream())
        G.sync(0, stream())
        ref = x.double().t() @ dz.double()
        assert float((dw.double() - ref).norm() / ref.norm()) <= 1e-6, (N, K, M)


# ---- the epilogue's gradient ----------------------------------------------------------------
def act_grad_ref(dy, z, act, p, seed, offset):
    v = dy.double()
    f = 1.0
    if p:
        f = torch.from_numpy(factors(*dy.shape, p, seed, offset)).cuda()
    s = slope64(z.double(), act) if act != "none" else torch.ones_like(v)
    ref = v * s * f
    # the slope's error: 2^-20 (1 + |z|), and that of the differences
    e = (v * f).abs() * ((2.0 ** -20 * (1 + z.double().abs()) if act not in ("none", "relu") else 0.0) + 2.0 ** -22)
    return ref, e


@pytest.mark.gpu
@pytest.mark.parametrize("act", ACT_NAMES)
@pytest.mark.parametrize("type", ["f16", "bf16"])
@pytest.mark.parametrize("size", [(1, 1), (1, 8), (3, 67), (37, 1003), (64, 64), (300, 520), (2500, 136), (5000, 300), (9000, 1024), (4500, 514)],
                         ids=str)
def test_act_grad(gemm, size, type, act):
    N, M = size
    t = ttype(type)
    dy, z = rand((N, M), t, 1), rand((N, M), t, 2, 2.0)
    z[0, 0] = 0.0
    for p in (0.0, 0.25):
        dz, db = torch.full_like(dy, float("nan")), torch.full((M,), float("nan"), device="cuda")
        G.act_grad(0, G.TYPES[type], dy, z if act != "none" else None, dz, db, N, M, act=G.ACTS[act], dropout_p=p,
                   seed=11, offset=12, stream=stream())
        G.sync(0, stream())
        ref, e = act_grad_ref(dy, z, act, p, 11, 12)
        if act == "gelu" or act == "gelu_tanh" or act == "silu":
            e = e + 1e-9 * dy.double().abs() * 2
        assert_close(dz, ref, e + half_step(ref, t) * 1.01, "dZ")
        # a sum of N values in f32, in any order: at most N roundings of the sum of magnitudes
        tol = e.sum(0) + ref.abs().sum(0) * (N * 2.0 ** -24) + 1e-30
        assert_close(db, ref.sum(0), tol, "dbias")
        only = torch.full((M,), float("nan"), device="cuda")
        G.act_grad(0, G.TYPES[type], dy, z, None, only, N, M, act=G.ACTS[act], dropout_p=p, seed=11, offset=12,
                   stream=stream())
        again = z.clone() if act != "none" else dy.clone()           # in place of Z (or of dY)
        G.act_grad(0, G.TYPES[type], dy if act != "none" else again, again, again, None, N, M, act=G.ACTS[act],
                   dropout_p=p, seed=11, offset=12, stream=stream())
        G.sync(0, stream())
        assert torch.equal(only, db) and torch.equal(again, dz)


@pytest.mark.gpu
def test_act_grad_strided_and_limits(gemm):
    N, M, t = 70, 200, torch.float16
    dy0, z0 = rand((N, M), t, 1), rand((N, M), t, 2)
    z0[3, 5], z0[4, 6], z0[5, 7] = float("inf"), float("-inf"), float("nan")
    for pad, shift in ((8, 8), (4, 4), (2, 2), (5, 3)):
        dy, z = put(dy0, M + pad, shift), put(z0, M + pad, shift)
        for act in ("relu", "gelu", "gelu_tanh", "silu"):
            buf, dz = strided((N, M), t, M + pad, shift, 7.0)
            G.act_grad(0, G.TYPES["f16"], dy, z, dz, None, N, M, act=G.ACTS[act], lddy=M + pad, ldz=M + pad,
                       lddz=M + pad, stream=stream())
            G.sync(0, stream())
            # the slopes' limits at the infinities are 1 and 0
            assert float(dz[3, 5]) == float(dy[3, 5]) and float(dz[4, 6]) == 0.0 and math.isnan(float(dz[5, 7]))
            ok = torch.isfinite(z0)
            ref, e = act_grad_ref(dy0, torch.where(ok, z0, torch.zeros_like(z0)), act, 0, 0, 0)
            got = torch.where(ok, dz, ref.to(t))
            assert_close(got, ref, e + 2e-9 + half_step(ref, t) * 1.01, act)
            dz.fill_(7.0)
            assert bool((buf == 7.0).all())


# ---- dropout ----------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("type", ["f16", "bf16"])
@pytest.mark.parametrize("size", [(1, 1), (1, 9), (3, 64), (33, 4104), (257, 131), (1000, 328)], ids=str)
def test_dropout(gemm, size, type):
    N, M = size
    t = ttype(type)
    x, r = rand((N, M), t, 1), rand((N, M), t, 2)
    x[0, 0] = float("inf")
    for p in (0.0, 0.1, 0.5, 1.0):
        f = torch.from_numpy(factors(N, M, p, 5, 2 ** 63 + 9)).cuda()
        for res in (None, r):
            y = torch.full_like(x, float("nan"))
            G.dropout(0, G.TYPES[type], x, y, N, M, p, 5, 2 ** 63 + 9, residual=res, stream=stream())
            G.sync(0, stream())
            v = torch.where(f == 0, torch.zeros_like(f), x.double() * f)
            ref = v if res is None else v + res.double()
            # in f32 the scale is off by 2^-24 and its product by 2^-24 more of |v|, which the sum may cancel
            # down from; the sum by 2^-24 of itself
            tol = torch.nan_to_num(v.abs(), posinf=0) * 2.0 ** -23 + ref.abs() * 2.0 ** -24
            assert_close(y, ref, tol + half_step(ref, t) * 1.01, f"p={p}")
            z = x.clone()                                             # in place
            G.dropout(0, G.TYPES[type], z, z, N, M, p, 5, 2 ** 63 + 9, residual=res, stream=stream())
            G.sync(0, stream())
            assert torch.equal(z, y)


@pytest.mark.gpu
def test_dropout_strided(gemm):
    N, M, t = 50, 136, torch.bfloat16
    x0, r0 = rand((N, M), t, 1), rand((N, M), t, 2)
    f = torch.from_numpy(factors(N, M, 0.3, 1, 2)).cuda()
    ref = x0.double() * f + r0.double()
    for pad, shift in ((8, 8), (8, 4), (4, 8), (2, 4), (6, 2), (3, 1)):
        buf, y = strided((N, M), t, M + pad, shift, 7.0)
        G.dropout(0, G.TYPES["bf16"], put(x0, M + pad, shift), y, N, M, 0.3, 1, 2, residual=put(r0, M + pad, shift),
                  ldx=M + pad, ldr=M + pad, ldy=M + pad, stream=stream())
        G.sync(0, stream())
        tol = (x0.double() * f).abs() * 2.0 ** -23 + ref.abs() * 2.0 ** -24      # as above
        assert_close(y, ref, tol + half_step(ref, t) * 1.01, "Y")
        y.fill_(7.0)
        assert bool((buf == 7.0).all())


# ---- past 32 bits --------------------------------------------------------------------------------
@pytest.mark.gpu
def test_offsets_past_32_bits(gemm):
    # 2.2e9 elements: the last rows lie behind 2^31 of them
    N, M, K, t = 270001, 8200, 24, torch.bfloat16
    x, w = rand((N, K), t, 1), rand((K, M), t, 2, K ** -0.5)
    y = torch.empty(N, M, dtype=t, device="cuda")
    G.linear(0, 1, x, w, y, N, K, M, act=G.ACTS["relu"], stream=stream())
    G.sync(0, stream())
    for lo, hi in ((0, 40), (N - 300, N)):
        z = x[lo:hi].double() @ w.double()
        v = act64(z, "relu")
        assert_close(y[lo:hi], v, 1.2 * product_error(x[lo:hi], w, K) + half_step(v, t) * 1.01, "Y")
    z = y[N - 300:].clone()
    db = torch.empty(M, device="cuda")
    G.act_grad(0, 1, y, y, y, db, N, M, act=G.ACTS["relu"], stream=stream())     # relu of a relu: y itself
    G.dropout(0, 1, y, y, N, M, 0.5, 3, 4, stream=stream())
    G.sync(0, stream())
    f = torch.from_numpy(factors(300, M, 0.5, 3, 4, first=N - 300)).cuda()
    assert torch.equal(y[N - 300:].double(), z.double() * f)
    dw = torch.empty(K, M, device="cuda")
    G.linear_dw(0, 1, x, y, dw, N, K, M, out_type=G.TYPES["f32"], stream=stream())
    G.sync(0, stream())
    ref = torch.zeros(K, M, dtype=torch.float64, device="cuda")
    mag = torch.zeros_like(ref)
    for i in range(0, N, 30000):
        a, b = x[i:i + 30000].double(), y[i:i + 30000].double()
        ref += a.t() @ b
        mag += a.abs().t() @ b.abs()
    assert_close(dw, ref, mag * ((512 / 16 + 16 + N / 512) * 2.0 ** -23) + half_step(ref, torch.float32), "dW")


# ---- together -----------------------------------------------------------------------------------
class Mlp:
    """x + D(W2 act(W1 x + b1) + b2), forward and backward through the C ABI."""

    def __init__(self, N, d, h, t, seed, act="gelu"):
        self.N, self.d, self.h, self.t, self.act = N, d, h, t, act
        self.ty = {torch.float16: 0, torch.bfloat16: 1}[t]
        self.w1, self.b1 = rand((d, h), t, seed, d ** -0.5), rand((h,), t, seed + 1, 0.1)
        self.w2, self.b2 = rand((h, d), t, seed + 2, h ** -0.5), rand((d,), t, seed + 3, 0.1)

    def empty(self, *shape, dtype=None):
        return torch.empty(*shape, dtype=dtype or self.t, device="cuda")

    def buffers(self):
        N, d, h = self.N, self.d, self.h
        f32 = torch.float32
        return dict(z=self.empty(N, h), a=self.empty(N, h), y=self.empty(N, d), dz2=self.empty(N, d),
                    da=self.empty(N, h), dz=self.empty(N, h), dx=self.empty(N, d),
                    db1=self.empty(h, dtype=f32), db2=self.empty(d, dtype=f32), dw1=self.empty(d, h, dtype=f32),
                    dw2=self.empty(h, d))

    def step(self, x, dy, o, p, seed, offset, offset_ptr=None):
        N, d, h, ty, st = self.N, self.d, self.h, self.ty, stream()
        drop = dict(dropout_p=p, seed=seed, offset=offset, offset_ptr=offset_ptr)
        G.linear(0, ty, x, self.w1, o["a"], N, d, h, bias=self.b1, act=G.ACTS[self.act], preact=o["z"], stream=st)
        G.linear(0, ty, o["a"], self.w2, o["y"], N, h, d, bias=self.b2, residual=x, stream=st, **drop)
        G.act_grad(0, ty, dy, None, o["dz2"], o["db2"], N, d, stream=st, **drop)
        G.linear_dw(0, ty, o["a"], o["dz2"], o["dw2"], N, h, d, stream=st)
        G.linear_dx(0, ty, o["dz2"], self.w2, o["da"], N, h, d, stream=st)
        G.act_grad(0, ty, o["da"], o["z"], o["dz"], o["db1"], N, h, act=G.ACTS[self.act], stream=st)
        G.linear_dw(0, ty, x, o["dz"], o["dw1"], N, d, h, out_type=G.TYPES["f32"], stream=st)
        G.linear_dx(0, ty, o["dz"], self.w1, o["dx"], N, d, h, residual=dy, stream=st)

    def reference(self, x, dy, p, seed, offset):
        leaves = [v.double().requires_grad_() for v in (x, self.w1, self.b1, self.w2, self.b2)]
        x, w1, b1, w2, b2 = leaves
        f = torch.from_numpy(factors(self.N, self.d, p, seed, offset)).cuda()
        y = x + f * (act64(x @ w1 + b1, self.act) @ w2 + b2)
        g = torch.autograd.grad(y, leaves, dy.double())
        return dict(zip(("y", "dx", "dw1", "db1", "dw2", "db2"), (y.detach(),) + g))


def assert_mlp(o, ref, t, what=""):
    # 2-norms: a result behind k chained roundings to t is off by at most about k steps; at most five here
    for name, v in ref.items():
        rel = float((o[name].double() - v).norm() / v.norm())
        assert rel <= 5 * torch.finfo(t).eps, f"{what}{name}: {rel:.3g}"


@pytest.mark.gpu
@pytest.mark.parametrize("type", ["f16", "bf16"])
@pytest.mark.parametrize("N", [1, 24, 300])
@pytest.mark.parametrize("act", ["gelu", "silu"])
def test_mlp_forward_and_backward(gemm, N, type, act):
    t = ttype(type)
    m = Mlp(N, 256, 520, t, 10, act)
    x, dy, o = rand((N, 256), t, 1), rand((N, 256), t, 2), m.buffers()
    m.step(x, dy, o, 0.1, 123, 456)
    G.sync(0, stream())
    assert_mlp(o, m.reference(x, dy, 0.1, 123, 456), t)


@pytest.mark.gpu
def test_mlp_captured_with_new_masks(gemm):
    # one captured step, replayed with the offset word rewritten in between: each replay has the masks of its offset
    t = torch.bfloat16
    m = Mlp(48, 264, 256, t, 20)
    x, dy, o = rand((48, 264), t, 1), rand((48, 264), t, 2), m.buffers()
    word = torch.zeros(1, dtype=torch.int64, device="cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        m.step(x, dy, o, 0.2, 9, 100, word)
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        m.step(x, dy, o, 0.2, 9, 100, word)
    seen = []
    for k in (0, 1, 7):
        word.fill_(k)
        g.replay()
        torch.cuda.synchronize()
        assert_mlp(o, m.reference(x, dy, 0.2, 9, 100 + k), t, f"replay with {k}: ")
        seen.append(o["y"].clone())
    assert not torch.equal(seen[0], seen[1])


@pytest.mark.gpu
def test_two_streams_and_repeats_agree(gemm):
    # the same call on two streams at once and again later: the same bits
    N, K, M, t = 96, 1032, 520, torch.float16
    x, w, dz = rand((N, K), t, 1), rand((K, M), t, 2, K ** -0.5), rand((N, M), t, 3)
    outs = []
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for s in streams * 2:
        with torch.cuda.stream(s):
            o = [torch.empty(N, M, dtype=t, device="cuda"), torch.empty(N, K, dtype=t, device="cuda"),
                 torch.empty(K, M, device="cuda"), torch.empty(M, device="cuda")]
            G.linear(0, 0, x, w, o[0], N, K, M, act=G.ACTS["silu"], stream=s.cuda_stream)
            G.linear_dx(0, 0, dz, w, o[1], N, K, M, stream=s.cuda_stream)
            G.linear_dw(0, 0, x, dz, o[2], N, K, M, out_type=G.TYPES["f32"], stream=s.cuda_stream)
            G.act_grad(0, 0, dz, None, None, o[3], N, M, stream=s.cuda_stream)
            outs.append(o)
    torch.cuda.synchronize()
    for o in outs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(o, outs[0]))


@pytest.mark.gpu
def test_first_calls_of_a_process_may_be_captured():
    # the kernels' one-time set-up needs no call before the capture
    import os
    import subprocess
    import sys
    code = f"""
import sys
sys.path.insert(0, {os.path.dirname(os.path.dirname(os.path.abspath(G.__file__)))!r})
import torch
from mlpgemm import lib as G
G.init(0)
t = torch.float16
x, w, dz = (torch.randn(*s, device="cuda").to(t) for s in ((40, 1000), (1000, 1336), (40, 1336)))
y, z = torch.empty_like(dz), torch.empty_like(dz)
dx, dw, db = torch.empty_like(x), torch.empty(1000, 1336, device="cuda"), torch.empty(1336, device="cuda")
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    s = torch.cuda.current_stream().cuda_stream
    G.linear(0, 0, x, w, y, 40, 1000, 1336, act=2, preact=z, dropout_p=0.1, seed=1, stream=s)
    G.act_grad(0, 0, dz, z, z, db, 40, 1336, act=2, stream=s)
    G.linear_dx(0, 0, z, w, dx, 40, 1000, 1336, stream=s)
    G.linear_dw(0, 0, x, z, dw, 40, 1000, 1336, out_type=2, stream=s)
    G.dropout(0, 0, y, y, 40, 1336, 0.5, 1, 2, stream=s)
g.replay()
torch.cuda.synchronize()
ref = x.double().t() @ z.double()
assert float((dw.double() - ref).norm() / ref.norm()) < 1e-6
print("captured")
"""
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "captured" in r.stdout, r.stderr[-2000:]


@pytest.mark.gpu
def test_fork_and_join_in_a_graph(gemm):
    # kernels set up early wait for everything before them: a long product on a forked stream, joined, then read
    N, K, M, t = 1536, 2048, 2048, torch.bfloat16
    x, w, x2 = rand((N, K), t, 1), rand((K, M), t, 2, K ** -0.5), rand((N, K), t, 3)
    a, b, c, y = (torch.zeros(N, M, dtype=t, device="cuda") for _ in range(4))
    s, side = torch.cuda.Stream(), torch.cuda.Stream()

    def step(wait=lambda: None):
        cur = torch.cuda.current_stream()
        G.linear(0, 1, x, w, a, N, K, M, stream=cur.cuda_stream)
        wait()
        side.wait_stream(cur)
        with torch.cuda.stream(side):
            G.linear(0, 1, x2, w, b, N, K, M, residual=a, stream=side.cuda_stream)
            wait()
            G.linear(0, 1, x2, w, b, N, K, M, residual=b, stream=side.cuda_stream)
            wait()
        G.dropout(0, 1, a, c, N, M, 0.0, 0, 0, stream=cur.cuda_stream)
        wait()
        cur.wait_stream(side)
        G.dropout(0, 1, c, y, N, M, 0.5, 1, 2, residual=b, stream=cur.cuda_stream)

    def run(call):
        for v in (a, b, c, y):
            v.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            call()
        torch.cuda.synchronize()
        return y.clone()

    ref = run(lambda: step(torch.cuda.synchronize))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        step()
    for _ in range(5):
        assert torch.equal(run(step), ref) and torch.equal(run(g.replay), ref)


@pytest.mark.gpu
def test_chained_calls_see_each_other(gemm):
    # a chain of small calls, each reading what the one before wrote, against the same chain with waits in between
    N, d, t = 33, 264, torch.float16
    w = rand((d, d), t, 1, d ** -0.5)
    x0 = rand((N, d), t, 2)

    def chain(wait):
        bufs = [x0.clone(), torch.empty_like(x0)]
        db = torch.empty(d, device="cuda")
        for i in range(40):
            a, b = bufs[i % 2], bufs[(i + 1) % 2]
            if i % 3 == 0:
                G.linear(0, 0, a, w, b, N, d, d, act=G.ACTS["silu"], residual=a, stream=stream())
            elif i % 3 == 1:
                G.dropout(0, 0, a, b, N, d, 0.1, i, 0, stream=stream())
            else:
                G.act_grad(0, 0, a, a, b, db, N, d, act=G.ACTS["gelu"], stream=stream())
            if wait:
                torch.cuda.synchronize()
        torch.cuda.synchronize()
        return bufs[0], db

    ref = chain(True)
    for _ in range(10):
        assert all(torch.equal(u, v) for u, v in zip(chain(False), ref))


@pytest.mark.gpu
def test_two_host_threads(gemm):
    import threading
    N, K, M, t = 64, 1000, 520, torch.bfloat16
    x, w = rand((N, K), t, 1), rand((K, M), t, 2, K ** -0.5)
    outs, errors = {}, []

    def work(i):
        try:
            s = torch.cuda.Stream()
            o = torch.empty(N, M, dtype=t, device="cuda")
            s.wait_stream(torch.cuda.default_stream())
            for _ in range(200):
                G.linear(0, 1, x, w, o, N, K, M, act=G.ACTS["gelu_tanh"], stream=s.cuda_stream)
            G.sync(0, s.cuda_stream)
            outs[i] = o
        except Exception as e:   # noqa: BLE001 - reported below
            errors.append(e)

    torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert not errors
    assert all(torch.equal(outs[i], outs[0]) for i in range(4))


# ---- refusals (no GPU needed: arguments are checked before the device) -----------------------------
P = 1 << 20   # stands for an aligned address; refused calls read nothing


def refused(call, *words):
    with pytest.raises(G.GemmError) as e:
        call()
    assert e.value.code == G.GEMM_ERR_ARGS, e.value
    for w in words:
        assert w in str(e.value), (w, str(e.value))


@pytest.mark.parametrize("kw,word", [
    (dict(type=2), "type"), (dict(type=-1), "type"), (dict(X=None), "null X"), (dict(W=None), "null W"),
    (dict(Y=None), "null Y"), (dict(N=0), "N=0"), (dict(K=-1), "K=-1"), (dict(M=(1 << 30) + 1), "M="),
    (dict(ldx=63), "X"), (dict(ldw=71), "W"), (dict(ldy=-72), "Y"), (dict(X=P + 1), "aligned"),
    (dict(Y=P + 1), "aligned"), (dict(bias=P + 1), "bias"), (dict(residual=P + 1), "residual"),
    (dict(residual=P, ldr=8), "residual"), (dict(Y=P), "same buffer"), (dict(preact=P), "same buffer"),
    (dict(residual=P + 8192, preact=P + 8192), "same buffer"), (dict(preact=P, ldz=8), "preact"), (dict(preact=P + 4096), "same buffer"),
    (dict(act=5), "activation"), (dict(act=-1), "activation"), (dict(dropout_p=1.5), "probability"),
    (dict(dropout_p=-0.1), "probability"), (dict(dropout_p=float("nan")), "probability"),
    (dict(offset_ptr=P + 4), "offset_ptr")])
def test_linear_refusals(kw, word):
    a = dict(type=0, X=P, W=P + 2048, Y=P + 4096, N=4, K=64, M=72)
    a.update(kw)
    refused(lambda: G.linear(0, **a), word)


def test_workspace_refusals():
    need = G.linear_workspace(G.OP_LINEAR, P, P + 2048, 4, 63, 72)
    assert need > 0
    for ws, n, word in ((None, 0, "workspace"), (P + 65536, need - 1, "workspace"), (P + 65536 + 8, need, "aligned")):
        refused(lambda: G.linear(0, 0, P, P + 2048, P + 4096, 4, 63, 72, workspace=ws, workspace_bytes=n), word)
        refused(lambda: G.linear_dw(0, 0, P, P + 2048, P + 4096, 4, 63, 72, workspace=ws, workspace_bytes=n), word)


def test_gradient_product_refusals():
    refused(lambda: G.linear_dx(0, 2, P, P, P, 4, 64, 72), "type")
    refused(lambda: G.linear_dx(0, 0, P, P, P + 64, 4, 64, 72, lddz=71), "dZ")
    refused(lambda: G.linear_dx(0, 0, P, P + 64, P, 4, 64, 72), "same buffer")
    refused(lambda: G.linear_dw(0, 0, P, P + 64, P + 64, 4, 64, 72), "same buffer")
    refused(lambda: G.linear_dx(0, 0, P, P, P + 64, 4, 64, 72, lddx=63), "dX")
    refused(lambda: G.linear_dx(0, 0, P, None, P, 4, 64, 72), "null W")
    refused(lambda: G.linear_dw(0, 0, P, P, P + 64, 4, 64, 72, out_type=1), "result type")
    refused(lambda: G.linear_dw(0, 1, P, P, P + 2, 4, 64, 72, out_type=2), "aligned")
    refused(lambda: G.linear_dw(0, 1, P, P, P + 64, 4, 64, 72, out_type=2, residual=P + 64, ldr=71), "residual")
    refused(lambda: G.linear_dw(0, 1, P, None, P, 4, 64, 72), "null dZ")


def test_act_grad_and_dropout_refusals():
    refused(lambda: G.act_grad(0, 0, P, None, P, P, 4, 8, act=2), "null Z")
    refused(lambda: G.act_grad(0, 0, P, P, None, None, 4, 8, act=2), "neither")
    refused(lambda: G.act_grad(0, 0, None, P, P, P, 4, 8, act=2), "null dY")
    refused(lambda: G.act_grad(0, 0, P, P, P, P + 2, 4, 8, act=2), "dbias")
    refused(lambda: G.act_grad(0, 0, P, P, P, P, 4, 8, act=9), "activation")
    refused(lambda: G.act_grad(0, 0, P, P, P, P, 0, 8), "N=0")
    refused(lambda: G.act_grad(0, 2, P, P, P, P, 4, 8), "type")
    refused(lambda: G.act_grad(0, 0, P, P, P, P, 4, 8, lddz=7), "dZ")
    refused(lambda: G.dropout(0, 0, P, P, 4, 8, 2.0, 0, 0), "probability")
    refused(lambda: G.dropout(0, 0, P, None, 4, 8, 0.5, 0, 0), "null Y")
    refused(lambda: G.dropout(0, 0, P, P, 4, 8, 0.5, 0, 0, ldx=7), "X")
    refused(lambda: G.dropout(0, 2, P, P, 4, 8, 0.5, 0, 0), "type")
    L = G.lib()
    assert L.gemm_dropout(0, 0, P, 0, None, 0, P, 0, 4, 8, None, None) == G.GEMM_ERR_ARGS


def test_good_arguments_need_the_device():
    if G.device_count() > 0:
        pytest.skip("a GPU is present")
    for call in (lambda: G.linear(0, 0, P, P, P + 4096, 4, 64, 72), lambda: G.linear_dx(0, 1, P, P, P + 4096, 4, 64, 72),
                 lambda: G.linear_dw(0, 1, P, P, P + 4096, 4, 64, 72, out_type=2),
                 lambda: G.act_grad(0, 0, P, P, P, P, 4, 8, act=1), lambda: G.dropout(0, 0, P, P, 4, 8, 0.5, 0, 0),
                 lambda: G.linear(99, 0, P, P, P + 4096, 4, 64, 72)):
        with pytest.raises(G.GemmError) as e:
            call()
        assert e.value.code == G.GEMM_ERR_INIT


def test_workspace_is_for_operands_the_tma_cannot_read():
    ws = G.linear_workspace
    assert ws(G.OP_LINEAR, P, P, 128, 1024, 2048) == 0
    assert ws(G.OP_LINEAR, P, P, 128, 1000, 2048, 1008, 2048) == 0
    assert ws(G.OP_LINEAR, P, P, 128, 1001, 2048) >= 128 * 1001 * 2          # X's rows
    assert ws(G.OP_LINEAR, P, P + 2, 128, 1024, 2048) >= 1024 * 2048 * 2     # W's base
    assert ws(G.OP_DX, P, P, 128, 1024, 1001) >= 128 * 1001 * 2 + 1024 * 1001 * 2
    assert ws(G.OP_DW, P, P, 128, 1001, 1024) >= 128 * 1001 * 2
    assert ws(G.OP_DW, P, P, 128, 1001, 1024, 1001, 0) < 128 * 1002 * 2 + 4096
    assert ws(3, P, P, 128, 1024, 2048) == 0 and ws(G.OP_LINEAR, None, P, 128, 1001, 2048) == 0
    assert ws(G.OP_LINEAR, P, P, 0, 1001, 2048) == 0


def test_structures_match_the_header():
    # the packed forms against C structures with the header's members (x86-64 layout)
    class Drop(ctypes.Structure):
        _fields_ = [("p", ctypes.c_double), ("seed", ctypes.c_uint64), ("offset", ctypes.c_uint64),
                    ("offset_ptr", ctypes.c_void_p)]

    class Epi(ctypes.Structure):
        _fields_ = [("bias", ctypes.c_void_p), ("residual", ctypes.c_void_p), ("ldr", ctypes.c_long),
                    ("preact", ctypes.c_void_p), ("ldz", ctypes.c_long), ("act", ctypes.c_int), ("dropout", Drop)]

    assert G.DROPOUT_ARGS.size == ctypes.sizeof(Drop) and G.EPILOGUE.size == ctypes.sizeof(Epi)
    e = Epi.from_buffer_copy(G.EPILOGUE.pack(1, 2, -3, 4, 5, 6, 0.75, 2 ** 64 - 1, 9, 10))
    assert (e.bias, e.residual, e.ldr, e.preact, e.ldz, e.act) == (1, 2, -3, 4, 5, 6)
    assert (e.dropout.p, e.dropout.seed, e.dropout.offset, e.dropout.offset_ptr) == (0.75, 2 ** 64 - 1, 9, 10)
    d = Drop.from_buffer_copy(G.DROPOUT_ARGS.pack(0.5, 7, 8, 0))
    assert (d.p, d.seed, d.offset, d.offset_ptr) == (0.5, 7, 8, None)
