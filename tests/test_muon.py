"""mg_orthogonalize and mg_muon_step against 64-bit evaluations.

Tolerances. The products round their operands to fp16 (half a step 2^-12 of a
value); how far that takes five steps from the exact iteration depends on the
matrix's spectrum, so the tests evaluate the same roundings in 64-bit
arithmetic on the test's matrix and allow 1.5 times that distance, plus 11 * 2^-11 / sqrt(s) of the
result's norm (s the smaller side): another summation order may round an entry
of B the other way, a step of 2^-11 of |B| <= 4.8 * 1.44 + 2.1 * 2.1 = 11, and s
by s entries do so independently. To that comes half a step of the output's
type on every entry, and 1e-5 for fp32 accumulation (K <= 4096 terms, 2^-24
each, grown by the steps as the fp16 roundings are).
"""
import ctypes

import numpy as np
import pytest

torch = pytest.importorskip("torch")

TYPES = {"f32": (0, torch.float32), "bf16": (1, torch.bfloat16), "f16": (2, torch.float16)}
A, B, C = 3.4445, -4.7750, 2.0315


def ok(mg, rc):
    assert rc == 0, mg.mg_last_error().decode()


def status(mg):
    torch.cuda.synchronize()
    st = ctypes.c_int(0)
    ok(mg, mg.mg_device_status(1, ctypes.byref(st)))
    return st.value


def newton_schulz(u, steps, rounded):
    """One matrix in 64 bits; rounded: the products' operands through fp16 at 2^10 scale, X through fp32."""
    def h(v):
        return (v * 1024).half().double() / 1024 if rounded else v

    u = u.double()
    n = u.norm()
    x = u / n if n > 0 else u
    flip = x.shape[0] > x.shape[1]
    x = x.t() if flip else x
    for _ in range(steps):
        x = x.float().double() if rounded else x
        g = h(h(x) @ h(x).t())
        x = A * x + h(B * g + C * (g @ g)) @ h(x)
    return x.t() if flip else x


def allowance(u, want, steps=5):
    near = newton_schulz(u, steps, True)
    return 1.5 * (near - want).norm() + (11 * 2.0 ** -11 / min(u.shape) ** 0.5 + 1e-5) * want.norm()


def matrix(gen, m, n, spectrum):
    u = torch.randn(m, n, generator=gen, device="cuda")
    if spectrum == "low rank":
        r = max(1, min(m, n) // 16)
        u = torch.randn(m, r, generator=gen, device="cuda") @ torch.randn(r, n, generator=gen, device="cuda") + 1e-3 * u
    if spectrum == "decaying":
        u = u * torch.logspace(0, -4, m, device="cuda")[:, None]
    return u


def workspace(mg, b, m, n):
    need = ctypes.c_size_t()
    ok(mg, mg.mg_muon_workspace(b, m, n, ctypes.byref(need)))
    return torch.full((need.value,), 0xFF, dtype=torch.uint8, device="cuda")  # NaN wherever it is read unwritten


def bad_orthogonalize():
    at = 1 << 20
    return dict(x=at, dtype=0, ld=64, stride=64 * 64, out=2 * at, out_dtype=1, ldo=64, out_stride=64 * 64, batch=2, rows=64, cols=64,
                steps=5, workspace=3 * at, bytes=1 << 30, stream=None)


def bad_step():
    at = 1 << 20
    return dict(master=at, grad=2 * at, momentum=3 * at, weights=4 * at, stride=64 * 64, batch=2, rows=64, cols=64, norms=5 * at, n=8,
                max_norm=0.5, lr=1e-3, scale=1.0, decay=0.9, nesterov=1, wd=0.0, steps=5, norm_out=None, workspace=6 * at,
                bytes=1 << 30, stream=None)


def test_bad_arguments_are_refused():
    """On the CPU: every check comes before any CUDA call."""
    import metalgym_b200

    lib = metalgym_b200.lib()
    need = ctypes.c_size_t()
    assert lib.mg_muon_workspace(1, 64, 64, None) == 1
    for b, m, n in ((0, 64, 64), (1, 0, 64), (1, 64, -1), (65536, 64, 64), (1, 65537, 64), (1, 64, 65537)):
        assert lib.mg_muon_workspace(b, m, n, ctypes.byref(need)) == 1
    assert lib.mg_muon_workspace(2, 64, 64, ctypes.byref(need)) == 0 and need.value > 0
    for spoil in (dict(x=None), dict(out=None), dict(dtype=3), dict(out_dtype=0), dict(out_dtype=3), dict(ld=63), dict(ldo=63),
                  dict(stride=4095), dict(out_stride=4095), dict(batch=0), dict(rows=0), dict(cols=0), dict(steps=0), dict(steps=17),
                  dict(workspace=None), dict(workspace=(3 << 20) + 8), dict(bytes=need.value - 1), dict(x=(1 << 20) + 2),
                  dict(out=(1 << 21) + 1)):
        assert lib.mg_orthogonalize(*dict(bad_orthogonalize(), **spoil).values()) == 1, spoil
        assert lib.mg_last_error()
    for spoil in (dict(master=None), dict(grad=None), dict(momentum=None), dict(weights=None), dict(stride=4095), dict(batch=0),
                  dict(rows=0), dict(cols=0), dict(n=-1), dict(norms=None), dict(norms=None, n=0), dict(norms=None, n=0, max_norm=0.0, norm_out=1 << 22),
                  dict(lr=float("nan")), dict(scale=float("inf")), dict(wd=float("nan")), dict(decay=float("nan")), dict(steps=0),
                  dict(workspace=None), dict(bytes=need.value - 1), dict(master=(1 << 20) + 2), dict(weights=(1 << 22) + 1)):
        assert lib.mg_muon_step(*dict(bad_step(), **spoil).values()) == 1, spoil
        assert lib.mg_last_error()


def test_misaligned_norms_are_refused():
    import metalgym_b200

    for spoil in (dict(norms=(1 << 22) + 2), dict(norm_out=(1 << 22) + 1)):
        assert metalgym_b200.lib().mg_muon_step(*dict(bad_step(), **spoil).values()) == 1, spoil
        assert b"aligned" in metalgym_b200.lib().mg_last_error()


SHAPES = [(1, 1, 1), (2, 1, 77), (1, 300, 1), (3, 5, 100), (2, 64, 64), (1, 65, 63), (4, 128, 512), (4, 512, 128), (2, 127, 129),
          (1, 129, 127), (1, 128, 1000), (2, 333, 1001), (1, 1001, 333), (1, 256, 1024), (2, 200, 40), (1, 640, 640), (9, 16, 24)]


@pytest.mark.gpu
@pytest.mark.parametrize("spectrum", ["normal", "low rank", "decaying"])
@pytest.mark.parametrize("batch,m,n", SHAPES)
def test_orthogonalize(mg, batch, m, n, spectrum):
    gen = torch.Generator(device="cuda").manual_seed(batch * 7 + m + n)
    u = torch.stack([matrix(gen, m, n, spectrum) * 10.0 ** (3 * i - 3) for i in range(batch)])
    space = workspace(mg, batch, m, n)
    for kind, out_kind, steps in (("f32", "bf16", 5), ("bf16", "f16", 5), ("f16", "bf16", 1), ("f32", "f16", 3)):
        code, dtype = TYPES[kind]
        if kind == "f16":
            u = u.clamp(-6e4, 6e4)
        x = torch.full((batch, m, n + 3), float("nan"), dtype=dtype, device="cuda")
        x[:, :, :n] = u
        out = torch.full((batch, m + 1, n + 5), 7.0, dtype=TYPES[out_kind][1], device="cuda")
        ok(mg, mg.mg_orthogonalize(x.data_ptr(), code, n + 3, m * (n + 3), out.data_ptr(), TYPES[out_kind][0], n + 5, (m + 1) * (n + 5), batch,
                                   m, n, steps, space.data_ptr(), space.numel(), None))
        assert status(mg) == 0
        assert (out[:, m] == 7).all() and (out[:, :, n:] == 7).all()
        half = torch.finfo(TYPES[out_kind][1]).eps / 2
        for i in range(batch):
            want = newton_schulz(x[i, :, :n], steps, False)
            off = (out[i, :m, :n].double() - want).norm()
            most = allowance(x[i, :, :n], want, steps) + half * want.norm() + 2.0 ** -25 * (m * n) ** 0.5
            assert off <= most, (kind, i, float(off / want.norm()))


@pytest.mark.gpu
@pytest.mark.parametrize("batch,m,n,steps", [(8, 1024, 1030, 2), (8, 1100, 1000, 2), (1, 1500, 2600, 2), (1, 2500, 1700, 2), (6, 520, 1300, 3)])
def test_matrices_of_many_tiles(mg, batch, m, n, steps):
    """Enough tiles for every tile shape and several to a CTA, edges inside them."""
    gen = torch.Generator(device="cuda").manual_seed(m * n + steps)
    x = torch.randn(batch, m, n, generator=gen, device="cuda")
    space = workspace(mg, batch, m, n)
    out = torch.empty(batch, m, n, dtype=torch.float16, device="cuda")
    ok(mg, mg.mg_orthogonalize(x.data_ptr(), 0, n, m * n, out.data_ptr(), 2, n, m * n, batch, m, n, steps, space.data_ptr(), space.numel(), None))
    assert status(mg) == 0
    for i in range(0, batch, max(1, batch - 1)):
        want = newton_schulz(x[i], steps, False)
        off = (out[i].double() - want).abs()
        assert off.norm() <= allowance(x[i], want, steps) + 2.0 ** -12 * want.norm()
        assert off.max() <= 0.05 * want.abs().max()  # no tile is wrong or missing


@pytest.mark.gpu
@pytest.mark.parametrize("batch,m,n,steps", [(2, 128, 512, 7), (1, 40, 200, 8), (3, 100, 30, 7), (1, 1, 9, 7), (1, 128, 128, 10), (2, 24, 24, 16)])
def test_many_steps_of_small_matrices(mg, batch, m, n, steps):
    """More steps than the one-kernel form takes: the tiled products at small sizes."""
    gen = torch.Generator(device="cuda").manual_seed(m * n + steps)
    x = torch.randn(batch, m, n, generator=gen, device="cuda")
    space = workspace(mg, batch, m, n)
    out = torch.empty(batch, m, n, dtype=torch.float16, device="cuda")
    ok(mg, mg.mg_orthogonalize(x.data_ptr(), 0, n, m * n, out.data_ptr(), 2, n, m * n, batch, m, n, steps, space.data_ptr(), space.numel(), None))
    assert status(mg) == 0
    for i in range(batch):
        want = newton_schulz(x[i], steps, False)
        assert (out[i].double() - want).norm() <= allowance(x[i], want, steps) + 2.0 ** -12 * want.norm()


@pytest.mark.gpu
@pytest.mark.parametrize("spectrum", ["normal", "low rank", "decaying"])
@pytest.mark.parametrize("batch,m,n", [(1, 128, 5000), (1, 3001, 20), (2, 64, 1024), (1, 1000, 65), (100, 16, 24), (160, 130, 17), (2, 100, 129), (1, 128, 128)])
def test_small_side_is_as_exact_as_fp32(mg, batch, m, n, spectrum):
    """A smaller side of at most 128 takes products of 22-bit operands: at most 16 of them in a row, each off by the
    operands' 2^-22 and by the cuts of the tensor cores' fp32 accumulator, 2^-23 in each of the 8 instructions of the
    leading parts, 16 * (2^-22 + 8 * 2^-23) = 1.9e-5 of the products' norms. The products are the powers of G, at most
    2, and P, whose norm is the largest ratio of a singular value of the result to that of X: the result is off by at
    most 1.9e-5 times that growth. The master weights show the update without a 16-bit rounding."""
    gen = torch.Generator(device="cuda").manual_seed(batch + m + n)
    grad = torch.stack([matrix(gen, m, n, spectrum) for _ in range(batch)])
    master, momentum = torch.zeros_like(grad), torch.zeros_like(grad)
    weights = torch.zeros(batch, m, n, dtype=torch.bfloat16, device="cuda")
    space = workspace(mg, batch, m, n)
    ok(mg, mg.mg_muon_step(master.data_ptr(), grad.data_ptr(), momentum.data_ptr(), weights.data_ptr(), m * n, batch, m, n, None, 0, 0.0, -1.0,
                           1.0, 0.0, 0, 0.0, 5, None, space.data_ptr(), space.numel(), None))
    assert status(mg) == 0
    for i in range(0, batch, max(1, batch // 5)):
        want = newton_schulz(grad[i], 5, False)
        x = grad[i].double() / grad[i].double().norm()
        left, size, right = torch.linalg.svd(x, full_matrices=False)
        growth = float((torch.einsum("ik,ij,kj->k", left, want, right) / size).max())
        assert (master[i].double() - want).norm() <= 16 * (2.0 ** -22 + 8 * 2.0 ** -23) * growth * want.norm()


def newton_schulz_parts(u, steps, gen):
    """The iteration in 64 bits with operands of two fp16 parts, X through fp32, and products whose fp32 accumulator is cut
    off after each of their 3 K / 16 instructions: 2^-24 of the sum a cut, and as noise 3 sqrt(3 K / 16) 2^-24 of an entry
    (or of the entries' root mean square: partial sums are no smaller), seven times what independent cuts of up to a step give."""
    def h(v):
        hi = (v * 1024).half().double()
        return (hi + (v * 1024 - hi).half().double()) / 1024

    def product(a, b):
        p, n = h(a) @ h(b), 3 * ((a.shape[1] + 15) // 16)
        size = p.abs().clamp(min=float(p.norm()) / p.numel() ** 0.5)
        return p * (1 - n * 2.0 ** -24) + 3 * n ** 0.5 * 2.0 ** -24 * size * torch.randn(p.shape, generator=gen, device=p.device, dtype=p.dtype)

    x = u.double() / u.double().norm()
    flip = x.shape[0] > x.shape[1]
    x = x.t() if flip else x
    for _ in range(steps):
        x = x.float().double()
        g = h(product(x, x.t()))
        x = A * x + product(B * g + C * product(g, g), x)
    return x.t() if flip else x


@pytest.mark.gpu
@pytest.mark.parametrize("spectrum", ["normal", "low rank", "decaying"])
@pytest.mark.parametrize("batch,m,n", [(1, 129, 1000), (2, 333, 1001), (1, 1001, 333), (1, 640, 640), (4, 512, 1030), (3, 200, 140), (1, 1100, 1000),
                                       (12, 1024, 1030)])
def test_larger_sides_are_as_exact_as_smaller_ones(mg, batch, m, n, spectrum):
    """Smaller sides above 128 take operands of 22 bits too: the master weights, which show the update without a 16-bit
    rounding, are off by at most 1.5 times the distance of the emulated roundings and 2^-20 of the update."""
    gen = torch.Generator(device="cuda").manual_seed(batch + m + n)
    grad = torch.stack([matrix(gen, m, n, spectrum) for _ in range(batch)])
    master, momentum = torch.zeros_like(grad), torch.zeros_like(grad)
    weights = torch.zeros(batch, m, n, dtype=torch.bfloat16, device="cuda")
    space = workspace(mg, batch, m, n)
    ok(mg, mg.mg_muon_step(master.data_ptr(), grad.data_ptr(), momentum.data_ptr(), weights.data_ptr(), m * n, batch, m, n, None, 0, 0.0, -1.0,
                           1.0, 0.0, 0, 0.0, 5, None, space.data_ptr(), space.numel(), None))
    assert status(mg) == 0
    for i in range(0, batch, max(1, batch - 1)):
        want = newton_schulz(grad[i], 5, False)
        near = newton_schulz_parts(grad[i], 5, gen)
        off = (master[i].double() - want).norm()
        assert off <= 1.5 * (near - want).norm() + 2.0 ** -20 * want.norm(), float(off / want.norm())


def newton_schulz_runs(u, steps, gen):
    """The form that smaller sides up to 128 take, with the roundings and cuts of newton_schulz_parts: three steps at a time on
    G = X X^T and P, the product of their polynomials of G; X between the runs in fp32."""
    def h(v, scale=1024):
        hi = (v * scale).half().double()
        return (hi + (v * scale - hi).half().double()) / scale

    def product(a, b):
        p, n = a @ b, 3 * ((a.shape[1] + 15) // 16)
        size = p.abs().clamp(min=float(p.norm()) / p.numel() ** 0.5)
        return p * (1 - n * 2.0 ** -24) + 3 * n ** 0.5 * 2.0 ** -24 * size * torch.randn(p.shape, generator=gen, device=p.device, dtype=p.dtype)

    x = u.double() / u.double().norm()
    flip = x.shape[0] > x.shape[1]
    x = (x.t() if flip else x).float().double()
    eye = torch.eye(x.shape[0], device=x.device, dtype=x.dtype)
    while steps:
        run = min(steps, 3)
        g, total = h(product(h(x), h(x).t())), None
        for step in range(run):
            q = h(A * eye + B * g + C * product(g, g))
            total = h(q if total is None else product(q, total.t()), 32)
            if step + 1 < run:
                g = h(product(q, h(product(q, g)).t()))
        x = product(total, h(x)).float().double()
        steps -= run
    return x.t() if flip else x


@pytest.mark.gpu
@pytest.mark.parametrize("steps", [2, 3, 4, 5, 6])
@pytest.mark.parametrize("rank", [1, 2, 8, 0])
@pytest.mark.parametrize("batch,m,n", [(1, 16, 200), (2, 64, 512), (1, 128, 512), (3, 512, 128), (1, 100, 3000), (1, 1500, 60), (1, 128, 128)])
def test_small_sides_of_any_rank_and_steps(mg, batch, m, n, rank, steps):
    """Matrices of few directions (0: as many as the smaller side, badly conditioned): the update is off by at most twice the
    distance of the emulated roundings and cuts and 2^-20 of it. (An emulation of one run of all the steps would allow 20
    times that at five steps and 100 times at six: G and P grow apart by a^2 a step in the directions that are hardly there.)"""
    gen = torch.Generator(device="cuda").manual_seed(batch + m + n + rank)
    r = rank or min(m, n)
    grad = torch.stack([torch.randn(m, r, generator=gen, device="cuda") @ torch.randn(r, n, generator=gen, device="cuda") for _ in range(batch)])
    master, momentum = torch.zeros_like(grad), torch.zeros_like(grad)
    weights = torch.zeros(batch, m, n, dtype=torch.bfloat16, device="cuda")
    space = workspace(mg, batch, m, n)
    ok(mg, mg.mg_muon_step(master.data_ptr(), grad.data_ptr(), momentum.data_ptr(), weights.data_ptr(), m * n, batch, m, n, None, 0, 0.0, -1.0,
                           1.0, 0.0, 0, 0.0, steps, None, space.data_ptr(), space.numel(), None))
    assert status(mg) == 0
    for i in range(0, batch, max(1, batch - 1)):
        want = newton_schulz(grad[i], steps, False)
        near = newton_schulz_runs(grad[i], steps, gen)
        off = (master[i].double() - want).norm()
        assert off <= 2 * (near - want).norm() + 2.0 ** -20 * want.norm(), float(off / want.norm())


@pytest.mark.gpu
@pytest.mark.parametrize("batch,m,n", [(1, 130, 300), (1, 333, 1001), (40, 161, 200), (3, 200, 1100), (1, 1030, 1500), (2, 129, 133), (1, 100, 700)])
def test_pieces_that_end_inside_a_warp(mg, batch, m, n):
    """Matrices whose last 32 x 32 pieces and mirrored pieces hold fewer rows than a warp has lanes, by every kind of
    product: the same bits every time, which are the result's (1.5 times the distance of the emulated roundings)."""
    gen = torch.Generator(device="cuda").manual_seed(m + n)
    x = torch.randn(batch, m, n, generator=gen, device="cuda")
    space = workspace(mg, batch, m, n)
    outs = [torch.empty(batch, m, n, dtype=torch.float16, device="cuda") for _ in range(20)]
    for out in outs:
        ok(mg, mg.mg_orthogonalize(x.data_ptr(), 0, n, m * n, out.data_ptr(), 2, n, m * n, batch, m, n, 3, space.data_ptr(), space.numel(), None))
    assert status(mg) == 0
    assert all(torch.equal(out, outs[0]) for out in outs)
    want = newton_schulz(x[0], 3, False)
    assert (outs[0][0].double() - want).norm() <= allowance(x[0], want, 3) + 2.0 ** -12 * want.norm()


@pytest.mark.gpu
def test_singular_values_come_near_one(mg):
    """Five steps take a well-spread spectrum into [0.6, 1.25] (the quintic's band [0.68, 1.21] and 0.3 % for the roundings)."""
    gen = torch.Generator(device="cuda").manual_seed(1)
    u = torch.randn(1, 256, 1024, generator=gen, device="cuda")
    space = workspace(mg, 1, 256, 1024)
    out = torch.empty(1, 256, 1024, dtype=torch.bfloat16, device="cuda")
    ok(mg, mg.mg_orthogonalize(u.data_ptr(), 0, 1024, 256 * 1024, out.data_ptr(), 1, 1024, 256 * 1024, 1, 256, 1024, 5, space.data_ptr(),
                               space.numel(), None))
    assert status(mg) == 0
    s = torch.linalg.svdvals(out[0].double())
    assert 0.6 < float(s.min()) and float(s.max()) < 1.25


@pytest.mark.gpu
@pytest.mark.parametrize("m,n", [(8, 40), (128, 512), (300, 200)])
def test_zero_tiny_huge_and_not_finite(mg, m, n):
    """A zero matrix gives zeros; matrices whose squares leave fp32's range their result; NaN stays in its matrix."""
    gen = torch.Generator(device="cuda").manual_seed(4)
    base = torch.randn(m, n, generator=gen, device="cuda")
    u = torch.stack([base * 0, base * 1e-30, base * 1e30, base, base])
    u[3, m // 2, n // 2] = float("nan")
    space = workspace(mg, 5, m, n)
    out = torch.empty(5, m, n, dtype=torch.float16, device="cuda")
    ok(mg, mg.mg_orthogonalize(u.data_ptr(), 0, n, m * n, out.data_ptr(), 2, n, m * n, 5, m, n, 5, space.data_ptr(), space.numel(), None))
    assert status(mg) == 0
    assert not out[0].any() and out[3].isnan().any() and not out[[0, 1, 2, 4]].isnan().any()
    want = newton_schulz(base, 5, False)
    for i in (1, 2, 4):
        assert (out[i].double() - want).norm() <= allowance(base, want) + 2.0 ** -12 * want.norm() + 2.0 ** -25 * (m * n) ** 0.5


@pytest.mark.gpu
@pytest.mark.parametrize("batch,m,n", [(2, 128, 512), (3, 512, 128), (1, 7, 9), (2, 333, 65), (1, 256, 1024)])
@pytest.mark.parametrize("nesterov,clip", [(1, 1), (0, 0), (1, 0)])
def test_muon_step(mg, batch, m, n, nesterov, clip):
    gen = torch.Generator(device="cuda").manual_seed(m + n)
    stride = m * n + 24  # the layers' other parameters lie between the matrices
    flat = [torch.randn(batch * stride, generator=gen, device="cuda") for _ in range(3)]
    master, grad, momentum = flat
    weights = master.bfloat16()
    before = [t.clone() for t in flat] + [weights.clone()]
    part = lambda t: torch.stack([t[i * stride: i * stride + m * n].reshape(m, n) for i in range(batch)])  # noqa: E731
    norms = torch.rand(5, generator=gen, device="cuda") * 100
    max_norm, lr, scale, decay, wd = 0.5, 2e-3, 3.0, 0.9, 0.1
    out_norm = torch.zeros(1, device="cuda")
    space = workspace(mg, batch, m, n)
    ok(mg, mg.mg_muon_step(master.data_ptr(), grad.data_ptr(), momentum.data_ptr(), weights.data_ptr(), stride, batch, m, n,
                           norms.data_ptr() if clip else None, 5 if clip else 0, max_norm if clip else 0.0, lr, scale, decay, nesterov, wd, 5,
                           out_norm.data_ptr() if clip else None, space.data_ptr(), space.numel(), None))
    assert status(mg) == 0
    g, mo, w = part(before[1]), part(before[2]), part(before[0])
    factor = np.float32(1)
    if clip:
        total = np.float32(0)
        for v in norms.cpu().numpy():
            total = np.float32(total + v)
        assert abs(out_norm.item() - total) <= 2.0 ** -21 * total
        norm = np.sqrt(np.float32(out_norm.item()))
        factor = np.float32(np.float32(max_norm) / np.float32(norm + np.float32(1e-6)))
    g = g * float(factor)
    mu = torch.tensor(decay, device="cuda")
    mo = mu * mo + g
    assert torch.equal(part(momentum), mo)  # fp32 operations in the same order
    u = g + mu * mo if nesterov else mo
    for i in range(batch):
        want = newton_schulz(u[i], 5, False)
        exact = w[i].double() * (1 - lr * wd) - lr * scale * want
        off = (part(master)[i].double() - exact).norm()
        assert off <= lr * scale * allowance(u[i], want) + 2.0 ** -22 * exact.norm()
    assert torch.equal(part(weights), part(master).bfloat16())
    # what lies between the matrices stays
    for t, b in zip((master, grad, momentum, weights), before):
        for i in range(batch):
            assert torch.equal(t[i * stride + m * n: (i + 1) * stride], b[i * stride + m * n: (i + 1) * stride])
    assert torch.equal(grad, before[1])


@pytest.mark.gpu
@pytest.mark.parametrize("m,n", [(64, 200), (200, 300)])
@pytest.mark.parametrize("offset", [0, 1, 3])
def test_buffers_off_vector_alignment(mg, m, n, offset):
    """Matrices whose first element, rows or distance from one to the next are not 16-byte aligned: the aligned call's bits."""
    gen = torch.Generator(device="cuda").manual_seed(offset + m)
    batch, results = 2, []
    grad = torch.randn(batch, m, n, generator=gen, device="cuda")
    master, momentum = torch.randn(batch, m, n, generator=gen, device="cuda"), torch.randn(batch, m, n, generator=gen, device="cuda")
    space = workspace(mg, batch, m, n)
    for shift, stride in ((0, m * n), (offset, m * n + offset)):
        def place(t, dtype=torch.float32):
            flat = torch.full((shift + batch * stride + 8,), 3.0, dtype=dtype, device="cuda")
            view = torch.as_strided(flat, (batch, m, n), (stride, n, 1), shift)
            view.copy_(t)
            return flat, view

        (fm, vm), (fg, vg), (fo, vo), (fw, vw) = place(master), place(grad), place(momentum), place(master, torch.bfloat16)
        ok(mg, mg.mg_muon_step(vm.data_ptr(), vg.data_ptr(), vo.data_ptr(), vw.data_ptr(), stride, batch, m, n, None, 0, 0.0, 0.01, 1.0, 0.9, 1,
                               0.0, 5, None, space.data_ptr(), space.numel(), None))
        out, view = place(master, torch.float16)
        ok(mg, mg.mg_orthogonalize(vw.data_ptr(), 1, n, stride, view.data_ptr(), 2, n, stride, batch, m, n, 5, space.data_ptr(), space.numel(), None))
        assert status(mg) == 0
        for flat in (fm, fg, fo, fw, out):  # what lies around the matrices stays
            assert (flat[:shift] == 3).all() and (flat[shift + (batch - 1) * stride + m * n:] == 3).all()
            assert (flat[shift + m * n: shift + stride] == 3).all()
        results.append([t.clone() for t in (vm, vo, vw, view)])
    for a, b in zip(*results):
        assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("m,n", [(128, 512), (300, 520)])
def test_captured_step_replays(mg, m, n):
    """A captured optimiser step replayed three times does what three calls do."""
    gen = torch.Generator(device="cuda").manual_seed(m)
    start = [torch.randn(2, m, n, generator=gen, device="cuda") for _ in range(3)]
    norm = torch.full((1,), 50.0, device="cuda")
    space = [workspace(mg, 2, m, n) for _ in range(2)]

    def buffers():
        master, grad, momentum = (t.clone() for t in start)
        return master, grad, momentum, master.bfloat16()

    def call(b, s, stream):
        ok(mg, mg.mg_muon_step(b[0].data_ptr(), b[1].data_ptr(), b[2].data_ptr(), b[3].data_ptr(), m * n, 2, m, n, norm.data_ptr(), 1, 0.5, 0.01,
                               1.0, 0.9, 1, 0.1, 5, None, s.data_ptr(), s.numel(), stream))

    plain, held = buffers(), buffers()
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        graph.capture_begin()
        call(held, space[1], side.cuda_stream)
        graph.capture_end()
        for _ in range(3):
            graph.replay()
    for _ in range(3):
        call(plain, space[0], None)
    torch.cuda.synchronize()
    assert status(mg) == 0
    for a, b in zip(plain, held):
        assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("m,n", [(64, 200), (200, 300)])
def test_step_after_a_refused_call(mg, m, n):
    """The error of a call that the runtime refused (host memory that no machine has) is that call's alone: the step behind
    it does what it does without it, and not the momentum alone."""
    gen = torch.Generator(device="cuda").manual_seed(m)
    start = [torch.randn(1, m, n, generator=gen, device="cuda") for _ in range(3)]
    space, results = workspace(mg, 1, m, n), []
    for refused in (False, True):
        master, grad, momentum = (t.clone() for t in start)
        weights = master.bfloat16()
        if refused:
            at = ctypes.c_void_p()
            assert mg.mg_host_alloc(1 << 60, ctypes.byref(at)) == 2 and mg.mg_last_error()
        ok(mg, mg.mg_muon_step(master.data_ptr(), grad.data_ptr(), momentum.data_ptr(), weights.data_ptr(), m * n, 1, m, n, None, 0, 0.0, 0.01,
                               1.0, 0.9, 1, 0.1, 5, None, space.data_ptr(), space.numel(), None))
        assert status(mg) == 0
        results.append((master, momentum, weights))
    for a, b in zip(*results):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_two_streams_two_workspaces_and_a_graph(mg):
    """Two calls at once with a workspace each, and a captured graph replayed beside one of them: the same bits as alone."""
    gen = torch.Generator(device="cuda").manual_seed(3)
    shapes = [(256, 768), (128, 512)]
    u = [torch.randn(1, m, n, generator=gen, device="cuda") for m, n in shapes]
    alone, spaces = [], [workspace(mg, 1, m, n) for m, n in shapes]

    def call(i, out, stream):
        m, n = shapes[i]
        ok(mg, mg.mg_orthogonalize(u[i].data_ptr(), 0, n, m * n, out.data_ptr(), 1, n, m * n, 1, m, n, 5, spaces[i].data_ptr(),
                                   spaces[i].numel(), stream))

    for i in range(2):
        out = torch.empty(shapes[i], dtype=torch.bfloat16, device="cuda")
        call(i, out, None)
        torch.cuda.synchronize()
        alone.append(out)
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [torch.zeros_like(o) for o in alone]
    torch.cuda.synchronize()
    with torch.cuda.stream(streams[1]):
        graph = torch.cuda.CUDAGraph()
        graph.capture_begin()
        call(1, outs[1], streams[1].cuda_stream)
        graph.capture_end()
    for _ in range(5):
        call(0, outs[0], streams[0].cuda_stream)
        with torch.cuda.stream(streams[1]):
            graph.replay()
    torch.cuda.synchronize()
    assert status(mg) == 0
    assert all(torch.equal(a, b) for a, b in zip(alone, outs))


@pytest.mark.gpu
def test_constrained_policy_iteration(mg):
    """The operators as one PPO iteration uses them: head GEMM, draw under masks and penalties, loss of the drawn actions,
    weight gradient, Muon step of the head. The gradient that comes back is the 64-bit formula's, the loss at the old policy
    has ratio 1 (approximate KL 0, nothing clipped), and the update moves each row's surrogate the right way."""
    gen = torch.Generator(device="cuda").manual_seed(6)
    rows, embed, actions = 512, 128, 512
    f = torch.randn(rows, embed, generator=gen, device="cuda").bfloat16()
    master = torch.randn(embed, actions, generator=gen, device="cuda") / embed ** 0.5
    w = master.bfloat16()
    logits = torch.empty(rows, actions, dtype=torch.bfloat16, device="cuda")
    ok(mg, mg.mg_gemm_bf16(f.data_ptr(), 0, embed, w.data_ptr(), 1, actions, rows, actions, embed, 0, logits.data_ptr(), actions, None, 0, 1, None))
    import metalgym_b200

    bits = torch.rand(rows, actions, generator=gen, device="cuda") < 0.5
    bits[5] = False
    value = (bits.reshape(rows, actions // 32, 32).long() << torch.arange(32, device="cuda")).sum(2)
    mask = torch.where(value > 0x7FFFFFFF, value - (1 << 32), value).int()
    history = torch.randint(0, actions, (rows, 40), generator=gen, device="cuda").int()
    rep = 1 + torch.rand(rows, generator=gen, device="cuda")
    c = metalgym_b200.LogitControls(mask=mask.data_ptr(), mask_stride=actions // 32, history=history.data_ptr(), history_stride=40,
                                    history_max=40, repetition=rep.data_ptr())
    words = torch.randint(1, 1 << 31, (rows,), generator=gen, device="cuda").int()
    action = torch.empty(rows, dtype=torch.int32, device="cuda")
    lp, ent = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
    ok(mg, mg.mg_logits_sample(logits.data_ptr(), 1, actions, ctypes.byref(c), words.data_ptr(), action.data_ptr(), lp.data_ptr(), ent.data_ptr(),
                               None, rows, actions, None))
    adv = torch.randn(rows, generator=gen, device="cuda")
    d, stats = torch.empty_like(logits), torch.empty(rows, 5, device="cuda")
    ok(mg, mg.mg_logits_policy_loss(logits.data_ptr(), 1, actions, ctypes.byref(c), action.data_ptr(), adv.data_ptr(), None, None, lp.data_ptr(),
                                    d.data_ptr(), actions, stats.data_ptr(), rows, actions, 0.2, 0.5, 0.01, 1.0 / rows, None))
    assert status(mg) == 0
    assert action[5] == -1 and bool((action >= 0).sum() == rows - 1)
    assert bits[torch.arange(rows, device="cuda"), action.clamp(min=0).long()][action >= 0].all()
    assert stats[:, 3].abs().max() < 1e-5 and not stats[:, 4].any()  # the same statistics, summed the same way
    torch.testing.assert_close(stats[:, 2], ent, rtol=1e-5, atol=1e-5)
    # the gradient by the formula
    x = logits.double()
    seen = torch.zeros(rows, actions, dtype=torch.bool, device="cuda").scatter_(1, history.long(), True)
    factor = torch.where(seen, torch.where(x > 0, 1 / rep.double()[:, None], rep.double()[:, None]), 1.0)
    l = (x * factor).masked_fill(~bits, -torch.inf)
    live = (action >= 0)[:, None]
    lsm = torch.log_softmax(torch.where(live, l, 0.0), 1)
    p = lsm.exp()
    h = torch.special.entr(p).sum(1, keepdim=True)
    hit = torch.nn.functional.one_hot(action.clamp(min=0).long(), actions)
    want = (-adv.double()[:, None] * (hit - p) + 0.01 * (p * h - torch.special.entr(p))) * factor / rows
    want = torch.where(live & bits, want, 0.0)
    # half a bf16 step of an entry, and 1e-5 of the row's terms for the fp32 statistics
    assert bool(((d.double() - want).abs() <= 2.0 ** -8 * want.abs() + 1e-5 * (adv.abs().double()[:, None] + 1) * factor / rows * (p + hit)).all())
    grad = torch.empty(embed, actions, device="cuda")
    ok(mg, mg.mg_gemm_bf16(f.data_ptr(), 1, embed, d.data_ptr(), 1, actions, embed, actions, rows, 4, grad.data_ptr(), actions, None, 0, 1, None))
    momentum, space = torch.zeros_like(grad), workspace(mg, 1, embed, actions)
    before = master.clone()
    norm = grad.square().sum().reshape(1)
    ok(mg, mg.mg_muon_step(master.data_ptr(), grad.data_ptr(), momentum.data_ptr(), w.data_ptr(), embed * actions, 1, embed, actions, norm.data_ptr(),
                           1, 0.5, 3e-4, 0.2 * actions ** 0.5, 0.95, 1, 0.0, 5, None, space.data_ptr(), space.numel(), None))
    assert status(mg) == 0
    # the update goes against the gradient: <O, G> is a sum of singular values
    assert float(((master - before) * grad).sum()) < 0
