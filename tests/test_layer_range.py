"""The MLP layer's operators at the ends of their ranges: long contractions, far values, wide tiles."""
import math

import pytest

import test_layer as L
from mlpgemm import lib as G
from test_layer import _torch  # noqa: F401 - sets test_layer.torch for GPU tests

torch = None


@pytest.fixture(autouse=True)
def _own_torch(request):
    global torch
    if request.node.get_closest_marker("gpu"):
        import torch as t
        torch = t


# ---- every kernel ---------------------------------------------------------------------------------
# (op, type, type of the result, N, K, M): what the shapes of test_layer.py do not reach (test_layer_plan.py checks)
KERNELS = [
    ("dx", "f16", "f16", 2136, 616, 7656), ("dx", "bf16", "bf16", 2101, 24, 4192), ("dx", "f16", "f16", 2061, 24, 696),
    ("dw", "bf16", "f32", 4625, 1, 24), ("dw", "bf16", "f32", 4489, 1035, 24), ("dw", "bf16", "f32", 1186, 3888, 313),
    ("dw", "f16", "f32", 4269, 65, 40), ("dw", "f16", "f32", 4520, 1056, 24), ("dw", "f16", "f32", 2080, 2184, 24),
    # contractions of several partial sums per CTA
    ("linear", "f16", "f16", 4156, 4416, 24), ("linear", "f16", "f16", 1, 32808, 24), ("linear", "f16", "f16", 137, 33632, 136),
    ("linear", "f16", "f16", 529, 35272, 24), ("linear", "f16", "f16", 1063, 35136, 24), ("linear", "f16", "f16", 2140, 16944, 24),
    ("linear", "bf16", "bf16", 4165, 33328, 24), ("linear", "bf16", "bf16", 1, 262872, 24),
    ("linear", "bf16", "bf16", 135, 268376, 136), ("linear", "bf16", "bf16", 532, 268793, 24),
    ("linear", "bf16", "bf16", 1032, 262224, 24), ("linear", "bf16", "bf16", 2063, 131344, 24),
    ("dx", "f16", "f16", 4336, 24, 4296), ("dx", "f16", "f16", 1, 24, 33176), ("dx", "f16", "f16", 129, 136, 37369),
    ("dx", "f16", "f16", 517, 24, 35424), ("dx", "f16", "f16", 1040, 24, 33552), ("dx", "f16", "f16", 2109, 24, 16608),
    ("dx", "bf16", "bf16", 4315, 24, 39032), ("dx", "bf16", "bf16", 1, 24, 263256), ("dx", "bf16", "bf16", 264, 24, 266456),
    ("dx", "bf16", "bf16", 522, 24, 279248), ("dx", "bf16", "bf16", 1100, 24, 266136), ("dx", "bf16", "bf16", 2106, 24, 136968),
    ("dw", "f16", "f16", 131699, 1, 24), ("dw", "f16", "f16", 48034, 1, 24), ("dw", "f16", "f16", 33008, 1088, 24),
    ("dw", "f16", "f16", 16760, 2072, 24), ("dw", "bf16", "bf16", 1087830, 1, 136), ("dw", "bf16", "bf16", 268775, 1, 24),
    ("dw", "bf16", "bf16", 283912, 1032, 24), ("dw", "bf16", "bf16", 164943, 2096, 24)]


@pytest.mark.gpu
@pytest.mark.parametrize("case", KERNELS, ids=str)
def test_every_kernel(gemm, case):
    # with a residual, in the result's own buffer and beside it: the same bits
    op, type, out, N, K, M = case
    t, o = L.ttype(type), L.ttype(out)
    a = L.rand(*{"linear": ((N, K), t, 1), "dx": ((N, M), t, 1), "dw": ((N, K), t, 1)}[op])
    b = L.rand(*{"linear": ((K, M), t, 2), "dx": ((K, M), t, 2), "dw": ((N, M), t, 2)}[op], scale=0.125)
    r = L.rand({"linear": (N, M), "dx": (N, K), "dw": (K, M)}[op], o, 3)
    kind, call = {"linear": (G.OP_LINEAR, G.linear), "dx": (G.OP_DX, G.linear_dx), "dw": (G.OP_DW, G.linear_dw)}[op]
    ws, wsb = L.workspace(kind, a, b, N, K, M)
    kw = dict(workspace=ws, workspace_bytes=wsb, stream=L.stream())
    if op == "dw":
        kw["out_type"] = G.TYPES[out]
    y, same = torch.full_like(r, float("nan")), r.clone()
    call(0, G.TYPES[type], a, b, y, N, K, M, residual=r, **kw)
    call(0, G.TYPES[type], a, b, same, N, K, M, residual=same, **kw)
    G.sync(0, L.stream())
    a, b = {"linear": lambda: (a, b), "dx": lambda: (a, b.t()), "dw": lambda: (a.t(), b)}[op]()
    depth, deep = a.shape[1], {"f16": 4096, "bf16": 32768, "f32": 512}[out]
    v = a.double() @ b.double() + r.double()
    # the cut of one partial sum (one unit of 2^-23 per step), and the additions of all
    e = (a.double().abs() @ b.double().abs()) * ((min(depth, deep) / 16 + 16) * 2.0 ** -23 + (depth / deep + 8) * 2.0 ** -24)
    L.assert_close(y, v, e + v.abs() * 2.0 ** -23 + L.half_step(v, o) * 1.01, op)
    assert torch.equal(same, y)


# ---- long contractions -------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("type,op,N,K,M", [
    ("f16", "linear", 4200, 131072, 40), ("f16", "linear", 5, 600000, 40), ("f16", "linear", 300, 70000, 264),
    ("f16", "linear", 4300, 4160, 264), ("f16", "dx", 4200, 40, 131072), ("f16", "dx", 20, 1032, 100000),
    ("f16", "dw", 1 << 20, 72, 88), ("f16", "dw", 120000, 72, 88), ("f16", "dw", 50001, 264, 24),
    ("bf16", "linear", 4200, 600000, 24), ("bf16", "dw", 600000, 136, 200), ("bf16", "dx", 9, 40, 300000),
    ("bf16", "spread", 4200, 600000, 24)])
def test_16_bit_sums_of_long_contractions(gemm, type, op, N, K, M):
    # All products are positive, so every bit that the tensor cores cut off makes a result smaller and nothing cancels.
    # A partial sum is at most 4096 deep for f16 and 32768 for bf16: a step for every 16 and 16 more inside one, each
    # cutting at most one unit of 2^-23; adding the partial sums rounds to nearest.
    # "spread" scales X's rows, so that the results lie on all sides of the type's steps.
    spread, op = op == "spread", "linear" if op == "spread" else op
    t = L.ttype(type)
    depth = {"linear": K, "dx": M, "dw": N}[op]
    deep = 4096 if type == "f16" else 32768
    g = torch.Generator(device="cuda").manual_seed(7)
    scale = 2.0 ** -4 if depth < 200000 else 2.0 ** -6

    def positive(*shape):
        return ((torch.rand(shape, generator=g, device="cuda") + 0.5) * scale).to(t)

    a = positive(*{"linear": (N, K), "dx": (N, M), "dw": (N, K)}[op])
    b = positive(*{"linear": (K, M), "dx": (K, M), "dw": (N, M)}[op])
    if spread:
        a *= torch.linspace(1, 2, N, device="cuda").to(t)[:, None]
    shape = {"linear": (N, M), "dx": (N, K), "dw": (K, M)}[op]
    out = torch.full(shape, float("nan"), dtype=t, device="cuda")
    ws, wsb = L.workspace({"linear": G.OP_LINEAR, "dx": G.OP_DX, "dw": G.OP_DW}[op], a, b, N, K, M)
    kw = dict(workspace=ws, workspace_bytes=wsb, stream=L.stream())
    if op == "linear":
        z = torch.full(shape, float("nan"), dtype=t, device="cuda")
        G.linear(0, G.TYPES[type], a, b, out, N, K, M, act=G.ACTS["relu"], preact=z, **kw)
    else:
        (G.linear_dx if op == "dx" else G.linear_dw)(0, G.TYPES[type], a, b, out, N, K, M, **kw)
    G.sync(0, L.stream())
    ref = torch.zeros(shape, dtype=torch.float64, device="cuda")
    for i in range(0, depth, 32768):
        s = slice(i, i + 32768)
        ref += {"linear": lambda: a[:, s].double() @ b[s].double(), "dx": lambda: a[:, s].double() @ b[:, s].double().t(),
                "dw": lambda: a[s].double().t() @ b[s].double()}[op]()
    cut = (min(deep, depth) / 16 + 16) * 2.0 ** -23 + (depth / deep + 8) * 2.0 ** -24
    L.assert_close(out, ref, L.half_step(ref, t) * 1.01 + ref * cut, op)
    # Over the whole matrix the roundings of the results cancel (five standard deviations of their mean) as far as the
    # values spread over the type's steps: rounding to steps s is a sawtooth of x, sum over k of (s / pi k) sin(2 pi k x / s)
    # up to signs, whose mean over normally distributed x of deviation d is at most the sum of (s / pi k)
    # exp(-2 (pi k d / s)^2) <= (s / pi) q / (1 - q), q = exp(-2 (pi d / s)^2), and never above s / 2
    off = float(((out.double() - ref) / ref).mean())
    step = 2.0 ** math.floor(math.log2(float(ref.max()))) * torch.finfo(t).eps
    q = math.exp(-2 * (math.pi * float(ref.std()) / step) ** 2)
    shared = min(step / 2, step / math.pi * q / (1 - q)) / float(ref.min())
    assert abs(off) <= cut + shared + 5 * torch.finfo(t).eps / 2 * ref.numel() ** -0.5, off
    if op == "linear":
        assert torch.equal(z, out)


@pytest.mark.gpu
def test_f32_dw_of_a_million_rows(gemm):
    # 2048 partial sums of 512 rows.  What each loses, some 5e-7 of it, has random signs and comes to as much of the sum.
    # An addition rounds off 0.29 units of the last place (root mean square), 0.29 * 0.72 * 2^-23 of a running sum that
    # grows with the root of its terms: sqrt(2048 / 2) times that is 8e-7.  Both together: 9.4e-7
    N, K, M = 1 << 20, 136, 88
    x, dz = L.rand((N, K), torch.bfloat16, 1), L.rand((N, M), torch.bfloat16, 2)
    dw = torch.empty(K, M, device="cuda")
    G.linear_dw(0, 1, x, dz, dw, N, K, M, out_type=G.TYPES["f32"], stream=L.stream())
    G.sync(0, L.stream())
    ref = x.double().t() @ dz.double()
    assert float((dw.double() - ref).norm() / ref.norm()) <= 1e-6


@pytest.mark.gpu
@pytest.mark.parametrize("type,K", [("f16", 8300), ("bf16", 66000)])
def test_epilogue_behind_several_partial_sums(gemm, type, K):
    # the pair kernel's whole epilogue where the sum is put together from three parts
    N, M, t = 4200, 520, L.ttype(type)
    x, w, b, r = L.rand((N, K), t, 1), L.rand((K, M), t, 2, K ** -0.5), L.rand((M,), t, 3), L.rand((N, M), t, 4)
    y, z = torch.empty(N, M, dtype=t, device="cuda"), torch.empty(N, M, dtype=t, device="cuda")
    ws, wsb = L.workspace(G.OP_LINEAR, x, w, N, K, M)
    for act in L.ACT_NAMES:
        G.linear(0, G.TYPES[type], x, w, y, N, K, M, bias=b, act=G.ACTS[act], residual=r, preact=z,
                 dropout_p=0.2, seed=3, offset=4, workspace=ws, workspace_bytes=wsb, stream=L.stream())
        G.sync(0, L.stream())
        ry, rz, ty, tz = L.linear_ref(x, w, b, r, act, 0.2, 3, 4)
        L.assert_close(y, ry, ty, "Y")
        L.assert_close(z, rz, tz, "Z")


# ---- activations over their whole range --------------------------------------------------------
def lower(z, act):
    """The factor of z in act(z), Phi(z) or a sigmoid, in 64 bits; and the exponent of the exp in it."""
    if act == "gelu":
        return 0.5 * torch.special.erfc(-z / 2 ** 0.5), z * z / 2
    u = (8 / math.pi) ** 0.5 * (z + 0.044715 * z ** 3) if act == "gelu_tanh" else z
    return torch.sigmoid(u), u


def act_and_slope(z, act):
    """act(z) and act'(z) in 64 bits with the errors that f32 arithmetic brings: 48 roundings and 1.5e-5 of approximation
    relative to the small side, and five roundings (2^-24) of the exponent, which pass to what falls with it, the small side.
    The slope's two terms cancel at its one zero.  Where the factor is below 2^-126 it
    counts as 0; the slope has it times 1 + |z u'| at most."""
    p, power = lower(z, act)
    small = lower(-z.abs(), act)[0]
    if act == "gelu":
        q = z * torch.exp(-z * z / 2) / (2 * math.pi) ** 0.5
        d = torch.ones_like(z)
    else:
        d = (8 / math.pi) ** 0.5 * (1 + 0.134145 * z * z) if act == "gelu_tanh" else torch.ones_like(z)
        q = z * p * lower(-z, act)[0] * d
    c, e = 48 * 2.0 ** -24, 1.5e-5 + 5 * power.abs() * 2.0 ** -24
    lost = 2.0 ** -126 * (1 + z.abs() * d)
    return z * p, (c * p + e * small) * z.abs() + lost, p + q, c * (p + q.abs()) + e * (small + q.abs()) + lost


@pytest.mark.gpu
@pytest.mark.parametrize("type", ["f16", "bf16"])
@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "silu"])
def test_activations_keep_their_digits(gemm, act, type):
    # every value of the type from 2^-12 to 1000 and its negative: results and slopes of the far negative side are tiny
    # and have to be as exact, relative to themselves, as any other
    t = L.ttype(type)
    bits = torch.arange(1 << 15, dtype=torch.int32, device="cuda").to(torch.int16).view(t)
    v = bits[(bits >= 2.0 ** -12) & (bits <= 1000)]
    v = torch.cat([v, -v, torch.zeros(8, dtype=t, device="cuda")])
    n = v.numel() // 8 * 8
    v = v[-n:].contiguous()
    z = v.double()
    y, ey, s, es = act_and_slope(z, act)
    one = torch.zeros(8, dtype=t, device="cuda")
    one[0] = 1
    for x, w, N, M in ((one[None], torch.stack([v] + [torch.zeros_like(v)] * 7), 1, n),             # a row of them
                       (v[:, None] * one[None], one[:, None] * torch.ones(8, device="cuda", dtype=t), n, 8)):
        out = torch.full((N, M), float("nan"), dtype=t, device="cuda")
        G.linear(0, G.TYPES[type], x, w, out, N, 8, M, act=G.ACTS[act], stream=L.stream())
        G.sync(0, L.stream())
        L.assert_close(out[0] if N == 1 else out[:, 0], y, L.half_step(y, t) * 1.01 + ey, act)
    dy, dz = torch.ones_like(v), torch.full_like(v, float("nan"))
    G.act_grad(0, G.TYPES[type], dy, v, dz, None, n // 8, 8, act=G.ACTS[act], stream=L.stream())
    G.sync(0, L.stream())
    L.assert_close(dz, s, L.half_step(s, t) * 1.01 + es, act + "'")


# ---- column sums of many rows --------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("N,M", [(270001, 8200), (1000003, 2051), (2000001, 24), (40000, 11008), (20000, 1000)])
def test_column_sums_of_many_rows(gemm, N, M):
    t = torch.bfloat16
    dy = torch.empty(N, M, dtype=t, device="cuda")
    z, dz, db = torch.empty_like(dy), torch.empty_like(dy), torch.full((M,), float("nan"), device="cuda")
    # positive values: the roundings of the additions (2^-24 each, 128 rows and then the runs one after the other) are
    # independent, so over all columns the 2-norm stays far below 1e-6
    for i in range(0, N, 50000):
        dy[i:i + 50000] = L.rand((min(50000, N - i), M), t, i + 1).abs()
        z[i:i + 50000] = L.rand((min(50000, N - i), M), t, i + 2)
    G.act_grad(0, 1, dy, z, dz, db, N, M, act=G.ACTS["relu"], stream=L.stream())
    G.sync(0, L.stream())
    ref = torch.zeros(M, dtype=torch.float64, device="cuda")
    for i in range(0, N, 50000):
        v = torch.where(z[i:i + 50000] > 0, dy[i:i + 50000], torch.zeros_like(dy[i:i + 50000]))
        assert torch.equal(dz[i:i + 50000], v)
        ref += v.double().sum(0)
    assert float((db.double() - ref).norm() / ref.norm()) <= 1e-6
    # equal values: the roundings go the same way; at most 128 rows, the runs (a slab's CTAs take 64 rows at a time or
    # more), and 8 + 8 + 16 additions that join threads and CTAs
    dy.fill_(0.1)
    row = torch.empty(M, device="cuda")
    for v in (0.3, 0.9, 1.3, 1.7, -0.4):
        z.fill_(v)
        G.act_grad(0, 1, dy, z, None, db, N, M, act=G.ACTS["gelu"], stream=L.stream())
        G.act_grad(0, 1, dy, z, None, row, 1, M, act=G.ACTS["gelu"], stream=L.stream())
        G.sync(0, L.stream())
        ref = row.double() * N
        assert float(((db.double() - ref) / ref).abs().max()) <= (128 + N / (128 * 64) + 32) * 2.0 ** -24, v


# ---- errors of other calls ----------------------------------------------------------------------
@pytest.mark.gpu
def test_an_earlier_calls_error_is_not_this_ones(gemm):
    # an allocation that the GPU cannot give fails by itself; the next call, here one that packs its operands, does not
    with pytest.raises(G.GemmError):
        G.DeviceBuffer(0, 1 << 50)
    N, K, M, t = 5, 33, 41, torch.float16
    x, w, y = L.rand((N, K), t, 1), L.rand((K, M), t, 2), torch.empty(N, M, dtype=t, device="cuda")
    ws, wsb = L.workspace(G.OP_LINEAR, x, w, N, K, M)
    assert wsb > 0
    G.linear(0, 0, x, w, y, N, K, M, workspace=ws, workspace_bytes=wsb, stream=L.stream())
    G.sync(0, L.stream())
    ry, _, ty, _ = L.linear_ref(x, w, None, None, "none", 0, 0, 0)
    L.assert_close(y, ry, ty, "Y")


@pytest.mark.gpu
def test_a_reported_error_is_over(gemm):
    # the same for the entry points that were there before: they ask cudaGetLastError after their launches
    src = torch.randn(64, 64, device="cuda")
    dst = torch.empty(64, 64, dtype=torch.uint8, device="cuda")
    with pytest.raises(G.GemmError):
        G.DeviceBuffer(0, 1 << 50)
    G.quantize(0, G.Q_E4M3, src, dst, None, 64, 64, stream=L.stream())
    G.sync(0, L.stream())
    back = dst.view(torch.float8_e4m3fn).double()
    assert bool(((back - src.double()).abs() <= src.double().abs() * 2.0 ** -4 + 2.0 ** -10).all())
