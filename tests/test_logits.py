"""Controlled logits (mg_logits_*) against plain numpy evaluations.

Tolerances. The controls are single rounded fp32 operations, so controlled
logits and the factors of their gradient are compared bit for bit (rounded
once to the output's type). The softmax statistics of n actions are sums of at
most K = n / 256 + 64 (or n / 32 + 64 below 1024 actions) fp32 terms an
accumulator, each term an exponential good to 2 ulp of an argument off by half
an ulp of its size D: relative error at most delta = (K + 4 + D) 2^-24. So
log-probabilities are off by at most delta + 2^-23 |value|, entropies (log s -
t / s, |t / s| <= D) by delta (1 + 2 D), and a gradient entry by the sums of its
terms times those errors, plus half a step of its type.
"""
import ctypes
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

TYPES = {"f32": (0, torch.float32), "bf16": (1, torch.bfloat16), "f16": (2, torch.float16)}
F = np.float32


def controls_struct(c, dev):
    """LogitControls over device copies (kept alive in `dev`) of the numpy arrays of c."""
    import metalgym_b200

    def at(key, dtype):
        if c.get(key) is None:
            return None
        dev[key] = torch.from_numpy(np.ascontiguousarray(c[key]).view(dtype)).cuda()
        return dev[key].data_ptr()

    s = metalgym_b200.LogitControls()
    s.mask, s.bias, s.history, s.history_len = (at("mask", np.int32), at("bias", np.float32), at("history", np.int32),
                                                at("history_len", np.int32))
    s.repetition, s.frequency, s.presence = (at(k, np.float32) for k in ("repetition", "frequency", "presence"))
    s.mask_stride = c["mask"].shape[1] if c.get("mask") is not None and c["mask"].shape[0] > 1 else 0
    s.bias_stride = c["bias"].shape[1] if c.get("bias") is not None and c["bias"].shape[0] > 1 else 0
    if c.get("history") is not None:
        s.history_stride, s.history_max = c["history"].shape[1], c.get("history_max", c["history"].shape[1])
    dev["struct"] = s
    return ctypes.byref(s)


def make_controls(rng, rows, actions, kinds):
    c = {}
    words = (actions + 31) // 32
    if "mask" in kinds or "shared_mask" in kinds:
        n = 1 if "shared_mask" in kinds else rows
        bits = rng.random((n, words * 32)) < rng.choice([0.1, 0.5, 0.95], size=(n, 1))
        bits[:, rng.integers(0, actions)] = True
        if n > 2:
            bits[1] = False  # nothing allowed
            bits[2] = False
            bits[2, actions - 1] = True  # one action left
        bits[:, actions:] = rng.random((n, words * 32 - actions)) < 0.5  # bits behind the last action mean nothing
        c["mask"] = np.packbits(bits.reshape(n, words, 32), axis=2, bitorder="little").view(np.uint32).reshape(n, words)
    if "bias" in kinds:
        c["bias"] = rng.standard_normal((1, actions)).astype(F)
    if "row_bias" in kinds:
        c["bias"] = rng.standard_normal((max(rows, 2), actions + 3)).astype(F)
    if "history" in kinds:
        h = int(rng.integers(1, 80))
        c["history"] = rng.integers(-3, min(actions, 12) + 3, (rows, h)).astype(np.int32)  # repeats, and entries that do not count
        c["history"][:, 0] = actions - 1
        c["history_len"] = rng.integers(-2, h + 4, rows).astype(np.int32)  # taken into [0, h]
        c["history_len"][0] = h
        c["repetition"] = (1 + rng.random(rows)).astype(F)
        c["frequency"] = rng.random(rows).astype(F)
        c["presence"] = rng.random(rows).astype(F)
    for k in ("no_repetition", "no_frequency", "no_presence"):
        if k in kinds:
            c.pop(k[3:], None)
    return c


def control_reference(x, c):
    """Controlled logits in fp32 (each operation rounded), whether allowed, occurrences."""
    rows, actions = x.shape
    n = np.zeros((rows, actions), np.int64)
    x = x.astype(F).copy()
    if c.get("history") is not None:
        h = c["history"]
        for r in range(rows):
            length = c.get("history_max", h.shape[1])
            if c.get("history_len") is not None:
                length = min(max(int(c["history_len"][r]), 0), length)
            for a in h[r, :length]:
                if 0 <= a < actions:
                    n[r, a] += 1
        one, zero = np.ones(rows, F), np.zeros(rows, F)
        rep, freq, pres = (c.get(k) if c.get(k) is not None else d for k, d in
                           (("repetition", one), ("frequency", zero), ("presence", zero)))
        with np.errstate(invalid="ignore", over="ignore"):
            y = np.where(x > 0, x / rep[:, None], x * rep[:, None]).astype(F)
            y = ((y - (freq[:, None] * n.astype(F)).astype(F)).astype(F) - pres[:, None]).astype(F)
        x = np.where(n > 0, y, x)
    if c.get("bias") is not None:
        x = (x + c["bias"][: rows if c["bias"].shape[0] > 1 else 1, :actions]).astype(F)
    ok = np.ones((rows, actions), bool)
    if c.get("mask") is not None:
        bits = np.unpackbits(c["mask"].view(np.uint8), axis=1, bitorder="little")[:, :actions].astype(bool)
        ok = np.broadcast_to(bits, (rows, actions)) if bits.shape[0] == 1 else bits[:rows]
        x = np.where(ok, x, F(-np.inf))
    return x, ok, n


def logits_of(rng, rows, ld, kind, scale=3.0):
    return (torch.from_numpy(rng.standard_normal((rows, ld)).astype(F)) * scale).to(TYPES[kind][1])


def ok(mg, rc):
    assert rc == 0, mg.mg_last_error().decode()


def status(mg):
    torch.cuda.synchronize()
    st = ctypes.c_int(0)
    ok(mg, mg.mg_device_status(1, ctypes.byref(st)))
    return st.value


SIZES = [(1, 1, 0), (3, 2, 62), (5, 31, 0), (4, 32, 0), (7, 33, 1), (70, 6, 58), (2, 1000, 7), (3, 1024, 0), (3, 1025, 2),
         (2, 8191, 1), (3, 8193, 0), (1, 16384, 0), (2, 50001, 0), (1, 131072, 0), (2, 40000, 8)]
KINDS = [(), ("mask",), ("history",), ("mask", "bias", "history"), ("shared_mask", "row_bias", "history", "no_frequency", "no_presence"),
         ("bias", "history", "no_repetition")]


# ------------------------------------------------------------------ refusals (CPU: every check comes before any CUDA call)


def good_call(name):
    """Arguments of a call that passes its checks but for what a test spoils (fake addresses: never launched)."""
    at = 1 << 20
    if name == "mg_logits_control":
        return dict(logits=at, dtype=1, ld=64, controls=None, out=2 * at, ldo=64, rows=4, actions=50, stream=None)
    if name == "mg_logits_control_backward":
        return dict(logits=at, dtype=1, ld=64, controls=None, d_out=2 * at, ldg=64, d_logits=3 * at, ldd=64, rows=4, actions=50, stream=None)
    if name == "mg_logits_sample":
        return dict(logits=at, dtype=1, ld=64, controls=None, rng=None, action=2 * at, log_prob=3 * at, entropy=None, value=None,
                    rows=4, actions=50, stream=None)
    return dict(logits=at, dtype=1, ld=64, controls=None, action=2 * at, adv=3 * at, adv_stats=None, ret=None, old=4 * at,
                d_logits=5 * at, ldd=64, stats=6 * at, rows=4, actions=50, clip=0.2, value_coef=0.5, entropy_coef=0.01,
                grad_scale=1.0, stream=None)


COMMON = [dict(logits=None), dict(dtype=3), dict(dtype=-1), dict(ld=49), dict(rows=0), dict(rows=-1), dict(actions=0),
          dict(actions=(1 << 18) + 1, ld=1 << 19, ldo=1 << 19, ldd=1 << 19, ldg=1 << 19), dict(logits=(1 << 20) + 1)]
OWN = {"mg_logits_control": [dict(out=None), dict(ldo=49), dict(out=(1 << 21) + 1), dict(out=1 << 20, ldo=72)],
       "mg_logits_control_backward": [dict(d_out=None), dict(d_logits=None), dict(ldg=49), dict(ldd=49),
                                      dict(d_logits=2 << 20, ldd=72), dict(d_logits=1 << 20, ldd=72)],
       "mg_logits_sample": [dict(action=None), dict(log_prob=None), dict(value=1 << 22, ld=50)],
       "mg_logits_policy_loss": [dict(action=None), dict(adv=None), dict(old=None), dict(stats=None), dict(d_logits=None),
                                 dict(ldd=49), dict(ret=1 << 22, ld=50), dict(ret=1 << 22, ldd=50), dict(clip=-0.1),
                                 dict(d_logits=1 << 20, ldd=72)]}
CONTROLS = [dict(mask=64, mask_stride=1), dict(mask=66, mask_stride=2), dict(bias=64, bias_stride=49), dict(bias=65),
            dict(repetition=64), dict(frequency=64), dict(presence=64), dict(history=64, history_max=0, history_stride=4),
            dict(history=64, history_max=(1 << 14) + 1, history_stride=1 << 15), dict(history=64, history_max=8, history_stride=7),
            dict(history=66, history_max=8, history_stride=8), dict(history=64, history_max=8, history_stride=8, frequency=65)]


@pytest.mark.parametrize("name", sorted(OWN))
def test_bad_arguments_are_refused(name):
    import metalgym_b200

    lib = metalgym_b200.lib()
    for spoil in COMMON + OWN[name]:
        args = good_call(name)
        args.update({k: v for k, v in spoil.items() if k in args})
        assert getattr(lib, name)(*args.values()) == 1, spoil
        assert lib.mg_last_error()
    for spoil in CONTROLS:
        c = metalgym_b200.LogitControls(**spoil)
        assert getattr(lib, name)(*dict(good_call(name), controls=ctypes.byref(c)).values()) == 1, spoil


@pytest.mark.parametrize("name", ["mg_logits_sample", "mg_logits_policy_loss"])
def test_misaligned_buffers_are_refused(name):
    import metalgym_b200

    lib = metalgym_b200.lib()
    keys = dict(mg_logits_sample=["rng", "action", "log_prob", "entropy", "value"],
                mg_logits_policy_loss=["action", "adv", "adv_stats", "ret", "old", "stats", "d_logits"])[name]
    for key in keys:
        args = good_call(name)
        args[key] = (1 << 22) + 1
        assert getattr(lib, name)(*args.values()) == 1, key
        assert b"aligned" in lib.mg_last_error()


def test_controls_layout_matches_the_header(tmp_path):
    """The ctypes structure has the C struct's size and offsets."""
    import subprocess
    from pathlib import Path

    import metalgym_b200

    fields = [f for f, _ in metalgym_b200.LogitControls._fields_]
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include "metalgym_b200.h"\nint main(void) {\n    printf("%zu\\n", sizeof(mg_logit_controls));\n'
                   + "".join(f'    printf("%zu\\n", offsetof(mg_logit_controls, {f}));\n' for f in fields) + "    return 0;\n}\n")
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-I", str(Path(__file__).resolve().parent.parent / "include"), str(src), "-o", str(exe)], check=True)
    got = [int(v) for v in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [ctypes.sizeof(metalgym_b200.LogitControls)] + [getattr(metalgym_b200.LogitControls, f).offset for f in fields]


# ------------------------------------------------------------------ control


@pytest.mark.gpu
@pytest.mark.parametrize("kind", sorted(TYPES))
@pytest.mark.parametrize("rows,actions,pad", SIZES)
def test_control_and_gradient(mg, rows, actions, pad, kind):
    code, dtype = TYPES[kind]
    ld, ldo = actions + pad, actions + (pad + 5) % 11
    for n, kinds in enumerate(KINDS):
        rng = np.random.default_rng(1000 * rows + actions + n)
        c = make_controls(rng, rows, actions, kinds)
        x = logits_of(rng, rows, ld, kind)
        want, allowed, count = control_reference(x[:, :actions].float().numpy(), c)
        if rows > 1 and "mask" in kinds:  # NaN, infinities and the type's lowest value in masked places have no effect
            bad = torch.tensor([math.nan, math.inf, -math.inf, torch.finfo(dtype).min]).to(dtype)
            hide = torch.from_numpy(~allowed.copy())
            x[:, :actions] = torch.where(hide, bad[torch.from_numpy(rng.integers(0, 4, allowed.shape))], x[:, :actions])
        dev = {}
        cs = controls_struct(c, dev)
        xd = x.cuda()
        out = torch.full((rows + 1, ldo), 7.0, dtype=dtype, device="cuda")
        ok(mg, mg.mg_logits_control(xd.data_ptr(), code, ld, cs, out.data_ptr(), ldo, rows, actions, None))
        dy = logits_of(rng, rows, ldo, kind, 1.0)
        if rows > 1 and "mask" in kinds:
            dy[:, :actions] = torch.where(hide, bad[torch.from_numpy(rng.integers(0, 4, allowed.shape))], dy[:, :actions])
        dyd = dy.cuda()
        dx = torch.full((rows + 1, ld), 7.0, dtype=dtype, device="cuda")
        ok(mg, mg.mg_logits_control_backward(xd.data_ptr(), code, ld, cs, dyd.data_ptr(), ldo, dx.data_ptr(), ld, rows, actions, None))
        assert status(mg) == 0
        torch.testing.assert_close(out[:rows, :actions].cpu(), torch.from_numpy(want).to(dtype), rtol=0, atol=0, equal_nan=True, msg=f"{kinds}")
        assert (out[rows] == 7).all() and (out[:, actions:] == 7).all() and (dx[rows] == 7).all() and (dx[:, actions:] == 7).all()
        g = dy[:, :actions].float().numpy()
        if c.get("repetition") is not None:
            rep = c["repetition"][:, None]
            with np.errstate(invalid="ignore"):
                g = np.where(count > 0, np.where(x[:, :actions].float().numpy() > 0, g / rep, g * rep), g).astype(F)
        g = np.where(allowed, g, F(0))
        torch.testing.assert_close(dx[:rows, :actions].cpu(), torch.from_numpy(g).to(dtype), rtol=0, atol=0, msg=f"{kinds}")
        # in place
        ok(mg, mg.mg_logits_control_backward(xd.data_ptr(), code, ld, cs, dyd.data_ptr(), ldo, dyd.data_ptr(), ldo, rows, actions, None))
        ok(mg, mg.mg_logits_control(xd.data_ptr(), code, ld, cs, xd.data_ptr(), ld, rows, actions, None))
        assert status(mg) == 0
        torch.testing.assert_close(dyd[:, :actions], dx[:rows, :actions], rtol=0, atol=0)
        torch.testing.assert_close(xd[:, :actions], out[:rows, :actions], rtol=0, atol=0, equal_nan=True)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("rows,actions,history", [(2048, 4096, 4096), (1500, 3000, 4100), (4096, 4096, 2048), (700, 1000, 16000)])
def test_gradient_of_a_history_without_repetition(mg, rows, actions, history, kind):
    """Frequency and presence penalties have derivative 1: the gradient passes through, masked or not, whatever the history's
    length; no table is made for it."""
    code, dtype = TYPES[kind]
    rng = np.random.default_rng(actions)
    g = torch.Generator(device="cuda").manual_seed(rows)
    x, dy = (torch.randn(rows, actions, generator=g, device="cuda").to(dtype) for _ in range(2))
    c = make_controls(rng, rows, actions, ("mask",))
    c["history"] = rng.integers(0, actions, (rows, history)).astype(np.int32)
    c["frequency"] = c["presence"] = np.full(rows, 0.5, F)
    dev = {}
    cs = controls_struct(c, dev)
    bits = np.unpackbits(c["mask"].view(np.uint8), axis=1, bitorder="little")[:, :actions].astype(bool)
    want = torch.where(torch.from_numpy(bits).cuda(), dy, torch.zeros((), dtype=dtype, device="cuda"))
    dx = torch.full((rows, actions), 7.0, dtype=dtype, device="cuda")
    ok(mg, mg.mg_logits_control_backward(x.data_ptr(), code, actions, cs, dy.data_ptr(), actions, dx.data_ptr(), actions, rows, actions, None))
    assert status(mg) == 0
    assert torch.equal(dx, want)


@pytest.mark.gpu
def test_longest_history_and_largest_action_set(mg):
    """The limits: 2^18 actions and 2^14 entries, one action taking every entry."""
    actions, h = 1 << 18, 1 << 14
    rng = np.random.default_rng(5)
    c = dict(history=np.stack([np.full(h, 131071), rng.integers(0, actions, h), rng.permutation(actions)[:h]]).astype(np.int32),
             repetition=np.full(3, 1.5, F), frequency=np.full(3, 0.25, F), presence=np.full(3, 0.5, F))
    x = logits_of(rng, 3, actions, "f32")
    want, _, _ = control_reference(x.numpy(), c)
    dev = {}
    xd, out = x.cuda(), torch.empty(3, actions, device="cuda")
    ok(mg, mg.mg_logits_control(xd.data_ptr(), 0, actions, controls_struct(c, dev), out.data_ptr(), actions, 3, actions, None))
    assert status(mg) == 0
    torch.testing.assert_close(out.cpu(), torch.from_numpy(want), rtol=0, atol=0)
    act, lp = torch.empty(3, dtype=torch.int32, device="cuda"), torch.empty(3, device="cuda")
    ok(mg, mg.mg_logits_sample(xd.data_ptr(), 0, actions, ctypes.byref(dev["struct"]), None, act.data_ptr(), lp.data_ptr(), None,
                               None, 3, actions, None))
    assert status(mg) == 0
    assert np.array_equal(act.cpu().numpy(), want.argmax(1))


# ------------------------------------------------------------------ draw


def delta(n, D):
    return ((n / 32 if n <= 1024 else n / 256) + 64 + 4 + D) * 2.0 ** -24


def next_word(w):
    w = w.astype(np.uint64)
    w ^= (w << np.uint64(13)) & np.uint64(0xFFFFFFFF)
    w ^= w >> np.uint64(17)
    return w ^ ((w << np.uint64(5)) & np.uint64(0xFFFFFFFF))


def race(words, actions):
    m = np.uint64(0xFFFFFFFF)
    h = (words[:, None] + np.arange(actions, dtype=np.uint64) * np.uint64(0x9E3779B9)) & m
    h ^= h >> np.uint64(16)
    h = (h * np.uint64(0x7FEB352D)) & m
    h ^= h >> np.uint64(15)
    h = (h * np.uint64(0x846CA68B)) & m
    h ^= h >> np.uint64(16)
    return -np.log1p(-(h.astype(np.float64) + 0.5) * 2.0 ** -32)


def softmax_reference(l):
    """log_softmax and entropy in 64 bits of rows that allow something (others: zeros)."""
    l = l.astype(np.float64)
    some = np.isfinite(l).any(1)
    top = np.where(some, l.max(1, initial=-np.inf), 0)[:, None]
    with np.errstate(divide="ignore", invalid="ignore"):
        lp = l - top - np.log(np.exp(l - top).sum(1, keepdims=True))
        p = np.exp(lp)
        h = -np.where(p > 0, p * lp, 0).sum(1)
    return lp, np.where(some, h, 0), some


@pytest.mark.gpu
@pytest.mark.parametrize("kind", sorted(TYPES))
@pytest.mark.parametrize("rows,actions,pad", SIZES)
def test_sample(mg, rows, actions, pad, kind):
    code, dtype = TYPES[kind]
    ld = actions + pad
    for n, kinds in enumerate(KINDS):
        rng = np.random.default_rng(77 * rows + actions + n)
        c = make_controls(rng, rows, actions, kinds)
        x = logits_of(rng, rows, ld, kind)
        l, allowed, _ = control_reference(x[:, :actions].float().numpy(), c)
        if "mask" in kinds and rows > 1:
            x[:, :actions] = torch.where(torch.from_numpy(~allowed.copy()), torch.tensor(math.nan).to(dtype), x[:, :actions])
        dev = {}
        cs = controls_struct(c, dev)
        xd = x.cuda()
        words = rng.integers(1, 1 << 32, rows, dtype=np.uint64)
        rd = torch.from_numpy(words.astype(np.uint32).view(np.int32).copy()).cuda()
        act = torch.full((rows + 1,), 99, dtype=torch.int32, device="cuda")
        lp, ent, val = (torch.full((rows + 1,), 99.0, device="cuda") for _ in range(3))
        for greedy in (False, True):
            ok(mg, mg.mg_logits_sample(xd.data_ptr(), code, ld, cs, None if greedy else rd.data_ptr(), act.data_ptr(), lp.data_ptr(),
                                       ent.data_ptr(), val.data_ptr() if pad else None, rows, actions, None))
            assert status(mg) == 0
            ref, h, some = softmax_reference(l)
            nw = next_word(words)
            with np.errstate(invalid="ignore"):
                key = l.astype(np.float64) if greedy else l - np.log(race(nw, actions))
            a = np.where(some, key.argmax(1), -1)
            assert np.array_equal(act.cpu().numpy()[:rows], a), (kinds, greedy)
            assert np.array_equal(rd.cpu().numpy().view(np.uint32), nw.astype(np.uint32))
            want = np.where(some, ref[np.arange(rows), np.maximum(a, 0)], 0)
            D = float(np.ptp(l[np.isfinite(l)])) if np.isfinite(l).any() else 0.0
            e = delta(actions, D)
            assert np.all(np.abs(lp.cpu().numpy()[:rows] - want) <= e + 2.0 ** -23 * (np.abs(want) + D)), kinds
            assert np.all(np.abs(ent.cpu().numpy()[:rows] - h) <= e * (1 + 2 * D) + 2.0 ** -22), kinds
            assert act[rows] == 99 and lp[rows] == 99 and ent[rows] == 99 and val[rows] == 99
            if pad:
                assert torch.equal(val[:rows], xd[:, actions].float())


@pytest.mark.gpu
def test_greedy_ties_take_the_lowest_index(mg):
    for actions in (2, 64, 1000, 20000):
        x = torch.zeros(5, actions, device="cuda").bfloat16()
        x[1, actions // 2:] = 1
        x[2, -1] = 1
        act, lp = torch.empty(5, dtype=torch.int32, device="cuda"), torch.empty(5, device="cuda")
        ok(mg, mg.mg_logits_sample(x.data_ptr(), 1, actions, None, None, act.data_ptr(), lp.data_ptr(), None, None, 5, actions, None))
        assert status(mg) == 0
        assert act.tolist() == [0, actions // 2, actions - 1, 0, 0]


@pytest.mark.gpu
@pytest.mark.parametrize("actions", [5, 2000])
def test_draws_follow_the_softmax(mg, actions):
    """Frequencies of 2^18 draws against p: each count within 6 standard deviations of its binomial."""
    rows = 1 << 18
    rng = np.random.default_rng(3)
    x = torch.from_numpy(rng.standard_normal((1, actions)).astype(F)).cuda()
    wide = x.expand(rows, actions).contiguous()
    words = torch.from_numpy(rng.integers(1, 1 << 32, rows, dtype=np.uint64).astype(np.uint32).view(np.int32).copy()).cuda()
    act, lp = torch.empty(rows, dtype=torch.int32, device="cuda"), torch.empty(rows, device="cuda")
    ok(mg, mg.mg_logits_sample(wide.data_ptr(), 0, actions, None, words.data_ptr(), act.data_ptr(), lp.data_ptr(), None, None, rows,
                               actions, None))
    assert status(mg) == 0
    p = torch.softmax(x[0].double(), 0).cpu().numpy()
    got = np.bincount(act.cpu().numpy(), minlength=actions)
    assert np.all(np.abs(got - rows * p) <= 6 * np.sqrt(rows * p * (1 - p)) + 1)


@pytest.mark.gpu
@pytest.mark.parametrize("offset", [0.0, 3000.0, -65536.0])
def test_draws_at_large_offsets(mg, offset):
    """A common offset of the logits (which fp32 still resolves) moves no draw: the definition's winner in 64 bits."""
    rng = np.random.default_rng(4)
    rows, actions = 400, 9000
    x = (rng.integers(-800, 800, (rows, actions)) / 128.0 + offset).astype(F)  # exact in fp32 at every offset
    words = rng.integers(1, 1 << 32, rows, dtype=np.uint64)
    xd, rd = torch.from_numpy(x).cuda(), torch.from_numpy(words.astype(np.uint32).view(np.int32).copy()).cuda()
    act, lp = torch.empty(rows, dtype=torch.int32, device="cuda"), torch.empty(rows, device="cuda")
    ok(mg, mg.mg_logits_sample(xd.data_ptr(), 0, actions, None, rd.data_ptr(), act.data_ptr(), lp.data_ptr(), None, None, rows, actions, None))
    assert status(mg) == 0
    want = (x.astype(np.float64) - np.log(race(next_word(words), actions))).argmax(1)
    assert np.array_equal(act.cpu().numpy(), want)


@pytest.mark.gpu
def test_nan_and_minus_infinity_at_allowed_actions(mg):
    x = torch.zeros(4, 40, device="cuda")
    x[0, 7] = math.nan
    x[1] = -math.inf
    x[2, :39] = -math.inf
    words = torch.arange(1, 5, dtype=torch.int32, device="cuda")
    act, lp, ent = torch.empty(4, dtype=torch.int32, device="cuda"), torch.empty(4, device="cuda"), torch.empty(4, device="cuda")
    ok(mg, mg.mg_logits_sample(x.data_ptr(), 0, 40, None, words.data_ptr(), act.data_ptr(), lp.data_ptr(), ent.data_ptr(), None, 4, 40, None))
    assert status(mg) == 0
    a = act.tolist()
    assert a[0] not in (-1, 7) and math.isnan(lp[0]) and math.isnan(ent[0])
    assert a[1] == -1 and lp[1] == 0 and ent[1] == 0
    assert a[2] == 39 and lp[2] == 0 and ent[2] == 0
    assert 0 <= a[3] < 40


@pytest.mark.gpu
@pytest.mark.parametrize("kind", sorted(TYPES))
@pytest.mark.parametrize("rows,actions,pad", [(24, 3, 0), (24, 40, 1), (24, 3000, 3), (8, 131072, 0), (3000, 1500, 5)])
def test_plus_infinity_at_allowed_actions(mg, kind, rows, actions, pad):
    """The largest l - log E is an allowed +infinity, the lowest of several: in the vector groups, at a row's edges, among
    the actions that occurred, beside NaN and masked infinities, as head GEMMs that overflow leave them. The statistics
    are NaN. Rows without one draw as ever."""
    code, dtype = TYPES[kind]
    rng = np.random.default_rng(actions)
    ld = actions + pad
    places = sorted({0, 1, 2, actions // 2, actions // 2 + 1, actions - 2, actions - 1, int(rng.integers(0, actions))} & set(range(actions)))
    for kinds in ((), ("mask", "bias", "history")):
        c = make_controls(rng, rows, actions, kinds)
        x = logits_of(rng, rows, ld, kind)
        for r in range(rows):
            if r % 5 == 4:
                continue
            at = rng.choice(places, size=1 + r % 5 % 3, replace=False) if len(places) > 2 else [places[r % len(places)]]
            if kinds and r % 2:
                at = [int(c["history"][r, 0])]  # one that occurred, where the history has an entry
            x[r, list(at)] = math.inf
            if r % 7 == 3:
                x[r, (int(at[0]) + 1) % actions] = math.nan
        l, _, _ = control_reference(x[:, :actions].float().numpy(), c)
        dev = {}
        cs = controls_struct(c, dev)
        xd = x.cuda()
        words = rng.integers(1, 1 << 32, rows, dtype=np.uint64)
        rd = torch.from_numpy(words.astype(np.uint32).view(np.int32).copy()).cuda()
        act = torch.empty(rows, dtype=torch.int32, device="cuda")
        lp, ent = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
        for greedy in (False, True):
            ok(mg, mg.mg_logits_sample(xd.data_ptr(), code, ld, cs, None if greedy else rd.data_ptr(), act.data_ptr(), lp.data_ptr(),
                                       ent.data_ptr(), None, rows, actions, None))
            assert status(mg) == 0
            key = l.astype(np.float64) if greedy else l - np.log(race(next_word(words), actions))
            key = np.where(np.isnan(key), -np.inf, key)  # a NaN is never drawn
            want = np.where((key > -np.inf).any(1), key.argmax(1), -1)
            assert np.array_equal(act.cpu().numpy(), want), (kinds, greedy)
            broken = (l == np.inf).any(1) | np.isnan(l).any(1)
            assert np.array_equal(np.isnan(lp.cpu().numpy()), broken) and np.array_equal(np.isnan(ent.cpu().numpy()), broken)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", sorted(TYPES))
@pytest.mark.parametrize("actions", [5, 40, 3000])
def test_logits_at_the_ends_of_the_type(mg, kind, actions):
    """Rows of the type's lowest number (a mask some programs write), of large offsets and of wide spreads: the softmax of
    equal logits is uniform whatever their size, and an entry far below the others has no weight."""
    code, dtype = TYPES[kind]
    low, high = torch.finfo(dtype).min, torch.finfo(dtype).max
    x = torch.full((6, actions), low, dtype=dtype)
    x[1, 2] = 0.0
    x[2] = high
    x[3] = low
    x[3, 1] = high
    x[4] = 1000.0
    x[4, :2] = 1008.0
    x[5, ::2] = -math.inf
    words = torch.arange(1, 7, dtype=torch.int32, device="cuda")
    xd = x.cuda()
    act, lp, ent = torch.empty(6, dtype=torch.int32, device="cuda"), torch.empty(6, device="cuda"), torch.empty(6, device="cuda")
    ok(mg, mg.mg_logits_sample(xd.data_ptr(), code, actions, None, words.data_ptr(), act.data_ptr(), lp.data_ptr(), ent.data_ptr(), None, 6,
                               actions, None))
    assert status(mg) == 0
    a = act.cpu().numpy()
    assert np.all((a >= 0) & (a < actions)) and a[1] == 2 and a[3] == 1 and a[5] % 2 == 1
    ref, h, _ = softmax_reference(x.float().numpy())
    e = delta(actions, 8.0)
    assert np.all(np.abs(lp.cpu().numpy() - ref[np.arange(6), a]) <= e + 2.0 ** -21)
    assert np.all(np.abs(ent.cpu().numpy() - h) <= e * 17 + 2.0 ** -21)
    d, st, z = torch.empty(6, actions, dtype=dtype, device="cuda"), torch.empty(6, 5, device="cuda"), torch.ones(6, device="cuda")
    ok(mg, mg.mg_logits_policy_loss(xd.data_ptr(), code, actions, None, act.data_ptr(), z.data_ptr(), None, None, lp.data_ptr(), d.data_ptr(),
                                    actions, st.data_ptr(), 6, actions, 0.2, 0.5, 0.0, 1.0, None))
    assert status(mg) == 0
    want = np.exp(ref) - (np.arange(actions) == a[:, None])
    assert np.all(np.abs(d.double().cpu().numpy() - want) <= 4 * e + torch.finfo(dtype).eps / 2 + 2.0 ** -20)


# ------------------------------------------------------------------ loss


def loss_reference(x, c, action, adv, adv_stats, ret, old, clip, vc, ec, scale):
    """The definition in 64 bits: gradient [rows][actions (+ 1)], stats, and a bound of the gradient's error."""
    rows, actions = len(action), x.shape[1] - (1 if ret is not None else 0)
    raw = x[:, :actions].astype(F)
    l, allowed, n = control_reference(raw, c)
    lp, h, _ = softmax_reference(l)
    D = float(np.ptp(l[np.isfinite(l)])) if np.isfinite(l).any() else 0.0
    e = delta(actions, D)
    g, st, tol = np.zeros((rows, x.shape[1])), np.zeros((rows, 5)), np.zeros((rows, x.shape[1]))
    for r in range(rows):
        a = int(action[r])
        if not 0 <= a < actions or not allowed[r, a] or not np.isfinite(l[r, a]):
            continue
        A = float(adv[r]) if adv_stats is None else (float(adv[r]) - float(adv_stats[0])) * float(adv_stats[1])
        ratio = math.exp(lp[r, a] - float(old[r]))
        one, two = ratio * A, min(max(ratio, 1 - clip), 1 + clip) * A
        slope = -A * ratio if one <= two else 0.0
        p = np.exp(lp[r])
        plp = np.where(p > 0, lp[r], 0)
        hit = np.arange(actions) == a
        f = np.ones(actions)
        if c.get("repetition") is not None:
            rep = float(c["repetition"][r])
            f = np.where(n[r] > 0, np.where(raw[r] > 0, 1 / rep, rep), 1.0)
        d = (slope * (hit - p) + ec * p * (plp + h[r])) * scale * f
        g[r, :actions] = np.where(allowed[r], d, 0)
        el = e * (1 + 2 * D) + 2.0 ** -22 * (1 + D + abs(float(old[r])))  # of a log-probability, and relative of the ratio
        tol[r, :actions] = np.abs(scale * f) * (abs(slope) * (hit + p) * 3 * el + abs(ec) * p * (np.abs(plp) + h[r] + 2) * 3 * el)
        vl = 0.0
        if ret is not None:
            err = float(x[r, actions]) - float(ret[r])
            vl = 0.5 * vc * err * err
            g[r, actions] = vc * err * scale
            tol[r, actions] = 2.0 ** -22 * abs(vc * scale) * (abs(float(x[r, actions])) + abs(float(ret[r])))
        st[r] = [-min(one, two), vl, h[r], float(old[r]) - lp[r, a], float(abs(ratio - 1) > clip)]
    return g, st, tol, e * (1 + 2 * D) + 2.0 ** -20


def loss_inputs(rng, x, c, rows, actions):
    l, allowed, _ = control_reference(x[:, :actions].astype(F), c)
    lp, _, some = softmax_reference(l)
    action = np.array([rng.choice(np.flatnonzero(allowed[r])) if allowed[r].any() else 0 for r in range(rows)], np.int32)
    if rows > 4:
        action[3] = -1  # padding
        action[4] = int(rng.integers(0, actions))  # perhaps masked
    old = np.where(some, lp[np.arange(rows), np.maximum(action, 0)], 0)
    # ratios on both sides of the clip, none within 1e-3 of its borders
    old = np.where(np.isfinite(old), old, 0) + rng.choice([-0.5, -0.1, 0.0, 0.1, 0.4], rows)
    return action, old.astype(F), rng.standard_normal(rows).astype(F)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", sorted(TYPES))
@pytest.mark.parametrize("rows,actions,pad", SIZES)
def test_policy_loss(mg, rows, actions, pad, kind):
    code, dtype = TYPES[kind]
    ld, ldd = actions + pad, actions + (pad + 9) % 13 + (1 if pad else 0)
    for n, kinds in enumerate(KINDS):
        rng = np.random.default_rng(31 * rows + actions + n)
        c = make_controls(rng, rows, actions, kinds)
        x = logits_of(rng, rows, ld, kind)
        with_ret, with_stats = pad > 0, n % 2 == 0
        columns = actions + (1 if with_ret else 0)
        xr = x.float().numpy()[:, :columns].copy()
        action, old, adv = loss_inputs(rng, xr, c, rows, actions)
        ret = rng.standard_normal(rows).astype(F) if with_ret else None
        adv_stats = np.array([0.1, 1.3], F) if with_stats else None
        scale = 1.0 / rows
        g, st, tol, el = loss_reference(xr, c, action, adv, adv_stats, ret, old, 0.2, 0.5, 0.03, scale)
        _, allowed, _ = control_reference(xr[:, :actions], c)
        if "mask" in kinds and rows > 1:
            x[:, :actions] = torch.where(torch.from_numpy(~allowed.copy()), torch.tensor(math.nan).to(dtype), x[:, :actions])
        dev = {}
        cs = controls_struct(c, dev)
        t = {k: torch.from_numpy(v).cuda() for k, v in dict(action=action, adv=adv, ret=ret, old=old, adv_stats=adv_stats).items() if v is not None}
        at = lambda k: t[k].data_ptr() if k in t else None  # noqa: E731
        xd = x.cuda()
        d = torch.full((rows + 1, ldd), 7.0, dtype=dtype, device="cuda")
        stats = torch.full((rows + 1, 5), 7.0, device="cuda")

        def call(out, ldo):
            ok(mg, mg.mg_logits_policy_loss(xd.data_ptr(), code, ld, cs, at("action"), at("adv"), at("adv_stats"), at("ret"), at("old"),
                                            out.data_ptr(), ldo, stats.data_ptr(), rows, actions, 0.2, 0.5, 0.03, scale, None))
            assert status(mg) == 0

        call(d, ldd)
        got = d[:rows, :columns].double().cpu().numpy()
        half = torch.finfo(dtype).eps / 2
        small = {"f32": 1e-38, "bf16": 1e-38, "f16": 2.0 ** -25}[kind]  # half the spacing of the smallest numbers
        off = np.abs(got - g) - (tol * (1 + 2 * half) + half * np.abs(g) + small)
        assert np.all(off <= 0), (kinds, off.max())
        sg = stats[:rows].double().cpu().numpy()
        bound = el * (1 + np.abs(st)) * 4 + 2.0 ** -20 * np.abs(st)
        ratio = np.exp(np.minimum(np.abs(st[:, 3:4]), 30))
        assert np.all(np.abs(sg - st) <= bound * ratio + 1e-7), (kinds, np.abs(sg - st).max(0))
        assert (d[rows] == 7).all() and (d[:, columns:] == 7).all() and (stats[rows] == 7).all()
        call(xd, ld)  # the gradient in the logits' place
        assert torch.equal(xd[:, :columns], d[:rows, :columns])


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("rows,actions,pad", [(640, 1000, 3), (1300, 2100, 1), (2400, 1100, 5)])
def test_many_rows(mg, monkeypatch, rows, actions, pad, kind):
    """So many rows that a warp takes each."""
    monkeypatch.setitem(globals(), "KINDS", [KINDS[0], KINDS[3]])
    test_control_and_gradient(mg, rows, actions, pad, kind)
    test_sample(mg, rows, actions, pad, kind)
    test_policy_loss(mg, rows, actions, pad, kind)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,actions,history", [(640, 1100, 90), (640, 1100, 700), (2800, 2000, 1240), (2800, 2000, 1244), (300, 200, 64), (300, 200, 65),
                                                  (3, 1, 90), (5, 6, 300), (8, 33, 2000)])
def test_tables_of_many_rows(mg, monkeypatch, rows, actions, history):
    """History tables on both sides of what sends rows to warps or CTAs: their size (100 KB for the eight of a CTA of warp
    teams: 1242 entries at 2000 actions) and their length for the rows, under every combination of penalties."""
    made = make_controls

    def longer(rng, rows, actions, kinds):
        c = made(rng, rows, actions, kinds)
        if "history" in c:
            c["history"] = rng.integers(-3, actions + 3, (rows, history)).astype(np.int32)
            c["history_len"] = rng.integers(-2, 40, rows).astype(np.int32)
            c["history_len"][:3] = history
        return c

    monkeypatch.setitem(globals(), "make_controls", longer)
    monkeypatch.setitem(globals(), "KINDS", KINDS[3:])
    test_control_and_gradient(mg, rows, actions, 3, "bf16")
    test_sample(mg, rows, actions, 3, "bf16")
    test_policy_loss(mg, rows, actions, 3, "bf16")


@pytest.mark.gpu
@pytest.mark.parametrize("rows,actions,pad", [(40, 20000, 3), (9, 8200, 1), (2, 262144, 0), (760, 33000, 1)])
def test_rows_in_parts(mg, monkeypatch, rows, actions, pad):
    """Rows of two, four and eight parts, and of two because they would not stay in L2."""
    monkeypatch.setitem(globals(), "KINDS", [KINDS[0], KINDS[3]])
    kind = "f32" if rows == 760 else "bf16"
    if rows < 760:
        test_sample(mg, rows, actions, pad, kind)
    test_policy_loss(mg, rows, actions, pad, kind)


@pytest.mark.gpu
def test_loss_gradient_against_differences(mg):
    """d(sum of row losses) / d(raw logit) by central differences of the 64-bit loss, penalties included."""
    rng = np.random.default_rng(9)
    rows, actions = 6, 7
    c = make_controls(rng, rows, actions, ("history", "bias"))
    x = rng.standard_normal((rows, actions)).astype(F)
    action, old, adv = loss_inputs(rng, x, c, rows, actions)
    action[3] = 2

    def total(v):
        one = {k: (w.astype(np.float64) if w.dtype == F else w) for k, w in c.items()}
        l = v.copy()
        n = control_reference(x, c)[2]
        l = np.where(n > 0, np.where(v > 0, v / one["repetition"][:, None], v * one["repetition"][:, None])
                     - one["frequency"][:, None] * n - one["presence"][:, None], v) + one["bias"]
        lp, h, _ = softmax_reference(l)
        ratio = np.exp(lp[np.arange(rows), action] - old)
        return float((-np.minimum(ratio * adv, np.clip(ratio, 0.8, 1.2) * adv) - 0.03 * h).sum())

    want = np.zeros((rows, actions))
    for i in np.ndindex(rows, actions):
        up, down = x.astype(np.float64), x.astype(np.float64)
        up[i] += 1e-5
        down[i] -= 1e-5
        want[i] = (total(up) - total(down)) / 2e-5
    dev = {}
    cs = controls_struct(c, dev)
    t = [torch.from_numpy(v).cuda() for v in (x, action, adv, old)]
    d, stats = torch.empty(rows, actions, device="cuda"), torch.empty(rows, 5, device="cuda")
    ok(mg, mg.mg_logits_policy_loss(t[0].data_ptr(), 0, actions, cs, t[1].data_ptr(), t[2].data_ptr(), None, None, t[3].data_ptr(),
                                    d.data_ptr(), actions, stats.data_ptr(), rows, actions, 0.2, 0.5, 0.03, 1.0, None))
    assert status(mg) == 0
    # differences: 1e-10 truncation and 1e-16 / 1e-5 cancellation; the kernel: 1e-5 of the terms, all below 10
    np.testing.assert_allclose(d.cpu().numpy(), want, rtol=0, atol=1e-4)


@pytest.mark.gpu
def test_loss_of_the_framework_head(mg):
    """Without controls, on the 64-column bf16 head: mg_policy_loss's gradient and statistics. Both round the same
    values to bf16 from arithmetic good to about 1e-6, so a gradient differs by at most one bf16 step."""
    rng = np.random.default_rng(2)
    rows, actions = 1000, 6
    x = logits_of(rng, rows, 64, "bf16").cuda()
    action = torch.from_numpy(rng.integers(0, actions, rows).astype(np.int32)).cuda()
    adv, ret = (torch.from_numpy(rng.standard_normal(rows).astype(F)).cuda() for _ in range(2))
    lp = torch.log_softmax(x[:, :actions].float(), 1)
    old = lp.gather(1, action.long()[:, None])[:, 0] + torch.from_numpy(rng.choice([-0.4, -0.1, 0.0, 0.1, 0.4], rows).astype(F)).cuda()
    a = [torch.zeros(rows, 64, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    s = [torch.zeros(rows, 5, device="cuda") for _ in range(2)]
    ok(mg, mg.mg_policy_loss(x.data_ptr(), action.data_ptr(), adv.data_ptr(), None, ret.data_ptr(), old.data_ptr(), a[0].data_ptr(),
                             s[0].data_ptr(), rows, actions, 0.2, 0.5, 0.01, None))
    ok(mg, mg.mg_logits_policy_loss(x.data_ptr(), 1, 64, None, action.data_ptr(), adv.data_ptr(), None, ret.data_ptr(), old.data_ptr(),
                                    a[1].data_ptr(), 64, s[1].data_ptr(), rows, actions, 0.2, 0.5, 0.01, 1.0 / rows, None))
    assert status(mg) == 0
    torch.testing.assert_close(a[1].float(), a[0].float(), rtol=2.0 ** -7, atol=1e-8)
    torch.testing.assert_close(s[1], s[0], rtol=1e-5, atol=1e-5)


@pytest.mark.gpu
def test_actions_outside_the_set_are_recorded(mg):
    x = torch.zeros(3, 10, device="cuda")
    action = torch.tensor([-1, 10, -7], dtype=torch.int32, device="cuda")
    z, d, st = torch.zeros(3, device="cuda"), torch.full((3, 10), 7.0, device="cuda"), torch.full((3, 5), 7.0, device="cuda")
    args = lambda n: (x.data_ptr(), 0, 10, None, action.data_ptr(), z.data_ptr(), None, None, z.data_ptr(), d.data_ptr(), 10,  # noqa: E731
                      st.data_ptr(), n, 10, 0.2, 0.5, 0.01, 1.0, None)
    ok(mg, mg.mg_logits_policy_loss(*args(1)))
    assert status(mg) == 0  # -1 is padding
    ok(mg, mg.mg_logits_policy_loss(*args(3)))
    assert status(mg) == 5  # the code of a bad action
    assert not d.any() and not st.any()


@pytest.mark.gpu
@pytest.mark.parametrize("actions", [9, 5000, 40000])
def test_loss_leaves_out_actions_of_logit_minus_infinity(mg, actions):
    """Rows whose action has the logit -inf (one of them with nothing else either), or was masked by the type's lowest
    number beside others: zeros in the first two, the ordinary loss in the third."""
    x = torch.zeros(3, actions + 1, device="cuda")
    x[0, 4] = -math.inf
    x[1, :actions] = -math.inf
    x[2, 5:actions] = torch.finfo(torch.float32).min
    action = torch.tensor([4, 2, 1], dtype=torch.int32, device="cuda")
    one, old = torch.ones(3, device="cuda"), torch.full((3,), -math.log(5.0), device="cuda")
    d, st = torch.full((3, actions + 1), 7.0, device="cuda"), torch.full((3, 5), 7.0, device="cuda")
    ok(mg, mg.mg_logits_policy_loss(x.data_ptr(), 0, actions + 1, None, action.data_ptr(), one.data_ptr(), None, one.data_ptr(), old.data_ptr(),
                                    d.data_ptr(), actions + 1, st.data_ptr(), 3, actions, 0.2, 0.5, 0.0, 1.0, None))
    assert status(mg) == 0
    assert not d[:2].any() and not st[:2].any()
    want = torch.zeros(actions + 1, device="cuda")
    want[:5] = 0.2  # p of the five, less 1 at the action; ratio 1, advantage 1; the value's 0.5 * (0 - 1)
    want[1] -= 1.0
    want[actions] = -0.5
    torch.testing.assert_close(d[2], want, rtol=0, atol=1e-6)
    torch.testing.assert_close(st[2], torch.tensor([-1.0, 0.25, math.log(5.0), 0.0, 0.0], device="cuda"), rtol=0, atol=2e-6)


@pytest.mark.gpu
@pytest.mark.parametrize("actions", [5, 2000])
def test_masked_gradients_are_zero_for_large_coefficients(mg, actions):
    """An entropy coefficient whose product with a masked action's logarithm overflows: zeros there all the same, and in
    a uniform row 0 at the others but for the roundings of p (ln p + H): 8 steps of the logarithm, times the coefficient."""
    mask = np.zeros((1, (actions + 31) // 32), np.uint32)
    mask[0, 0] = 0b1011
    dev = {}
    cs = controls_struct(dict(mask=mask), dev)
    x = torch.zeros(2, actions, device="cuda")
    action, zero = torch.tensor([0, 3], dtype=torch.int32, device="cuda"), torch.zeros(2, device="cuda")
    d, st = torch.full((2, actions), 7.0, device="cuda"), torch.empty(2, 5, device="cuda")
    ok(mg, mg.mg_logits_policy_loss(x.data_ptr(), 0, actions, cs, action.data_ptr(), zero.data_ptr(), None, None, zero.data_ptr(),
                                    d.data_ptr(), actions, st.data_ptr(), 2, actions, 0.2, 0.5, 1e9, 1.0, None))
    assert status(mg) == 0
    allowed = torch.zeros(actions, dtype=torch.bool, device="cuda")
    allowed[[0, 1, 3]] = True
    assert not d[:, ~allowed].any()
    assert (d[:, allowed].abs() <= 1e9 * 8 * 2.0 ** -23 * math.log(3.0)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("rows,actions", [(3, 50), (2, 4000)])
def test_history_without_lengths_and_wider_rows(mg, rows, actions):
    """history_len NULL takes history_max entries of every row, of rows that lie further apart than that."""
    rng = np.random.default_rng(actions)
    wide = rng.integers(0, actions, (rows, 30)).astype(np.int32)
    c = dict(history=wide, history_max=11, frequency=np.full(rows, 0.5, F))
    x = logits_of(rng, rows, actions, "f32")
    want, _, count = control_reference(x.numpy(), c)
    assert count.sum() == 11 * rows
    dev = {}
    xd, out = x.cuda(), torch.empty(rows, actions, device="cuda")
    ok(mg, mg.mg_logits_control(xd.data_ptr(), 0, actions, controls_struct(c, dev), out.data_ptr(), actions, rows, actions, None))
    assert status(mg) == 0
    torch.testing.assert_close(out.cpu(), torch.from_numpy(want), rtol=0, atol=0)


@pytest.mark.gpu
def test_rows_past_32_bit_offsets(mg):
    """The last row of a tensor of more than 2^32 bytes (and 2^31 elements)."""
    ld = 1 << 21
    rows, actions = 1100, 500
    x = torch.empty(rows, ld, dtype=torch.bfloat16, device="cuda")
    x[:, :actions] = torch.randn(rows, actions, device="cuda")
    act, lp = torch.empty(rows, dtype=torch.int32, device="cuda"), torch.empty(rows, device="cuda")
    ok(mg, mg.mg_logits_sample(x.data_ptr(), 1, ld, None, None, act.data_ptr(), lp.data_ptr(), None, None, rows, actions, None))
    assert status(mg) == 0
    best = x[:, :actions].float()
    assert torch.equal(best.gather(1, act.long()[:, None])[:, 0], best.amax(1))


@pytest.mark.gpu
def test_stream_capture_and_repeat(mg):
    """On a side stream and inside a captured graph, the same bits; a replay advances the words."""
    rng = np.random.default_rng(8)
    rows, actions = 37, 3001
    c = make_controls(rng, rows, actions, ("mask", "bias", "history"))
    dev = {}
    cs = controls_struct(c, dev)
    x = logits_of(rng, rows, actions, "bf16").cuda()
    first = torch.arange(1, rows + 1, dtype=torch.int32, device="cuda")

    def fresh():
        return first.clone(), torch.empty(rows, dtype=torch.int32, device="cuda"), torch.empty(rows, device="cuda")

    def call(bufs, stream):
        w, a, lp = bufs
        ok(mg, mg.mg_logits_sample(x.data_ptr(), 1, actions, cs, w.data_ptr(), a.data_ptr(), lp.data_ptr(), None, None, rows, actions, stream))

    plain = fresh()
    call(plain, None)
    torch.cuda.synchronize()
    one = [t.clone() for t in plain]
    call(plain, None)
    torch.cuda.synchronize()
    captured = fresh()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        graph.capture_begin()
        call(captured, side.cuda_stream)
        graph.capture_end()
        graph.replay()
    torch.cuda.synchronize()
    for got, want in zip(captured, one):
        assert torch.equal(got, want)
    graph.replay()
    torch.cuda.synchronize()
    for got, want in zip(captured, plain):
        assert torch.equal(got, want)
    assert status(mg) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("rows,actions", [(300, 70), (40, 9000), (3, 60000)])
def test_two_calls_at_once_and_a_repeat(mg, rows, actions):
    """Loss and draw of the same logits on two streams together, twice: the bits of the calls made one after the other."""
    rng = np.random.default_rng(rows)
    c = make_controls(rng, rows, actions, ("mask", "bias", "history"))
    dev = {}
    cs = controls_struct(c, dev)
    xn = logits_of(rng, rows, actions, "bf16")
    action, old, adv = loss_inputs(rng, xn.float().numpy(), c, rows, actions)
    x = xn.cuda()
    t = [torch.from_numpy(v).cuda() for v in (action, adv, old)]
    first = torch.arange(1, rows + 1, dtype=torch.int32, device="cuda")

    def loss(stream):
        d, st = torch.zeros_like(x), torch.zeros(rows, 5, device="cuda")
        torch.cuda.synchronize()
        return d, st, lambda: ok(mg, mg.mg_logits_policy_loss(
            x.data_ptr(), 1, actions, cs, t[0].data_ptr(), t[1].data_ptr(), None, None, t[2].data_ptr(), d.data_ptr(), actions, st.data_ptr(),
            rows, actions, 0.2, 0.5, 0.01, 1.0, stream))

    def draw(stream):
        w, a, lp = first.clone(), torch.zeros(rows, dtype=torch.int32, device="cuda"), torch.zeros(rows, device="cuda")
        torch.cuda.synchronize()
        return w, a, lp, lambda: ok(mg, mg.mg_logits_sample(x.data_ptr(), 1, actions, cs, w.data_ptr(), a.data_ptr(), lp.data_ptr(), None, None,
                                                            rows, actions, stream))

    one, two = loss(None), draw(None)
    one[-1]()
    torch.cuda.synchronize()
    two[-1]()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(2):
        three, four = loss(streams[0].cuda_stream), draw(streams[1].cuda_stream)
        three[-1]()
        four[-1]()
        torch.cuda.synchronize()
        for a, b in zip((*one[:-1], *two[:-1]), (*three[:-1], *four[:-1])):
            assert torch.equal(a, b)
    assert status(mg) == 0


@pytest.mark.gpu
def test_documented_example_runs(mg):
    """The Python block of the integration guide: it runs, draws only allowed actions, and its gradient is finite."""
    from pathlib import Path

    text = (Path(__file__).resolve().parent.parent / "INTEGRATION.md").read_text()
    blocks = [b.split("```")[0] for b in text.split("```python")[1:]]
    block = next(b for b in blocks if "mg_logits_sample" in b)
    names = {}
    exec(compile(block, "example", "exec"), names)
    assert status(mg) == 0
    assert not (names["action"] % 2).any() and (names["action"] >= 0).all()
    assert names["grad"].isfinite().all() and names["grad"].any() and names["master"].isfinite().all()
    assert torch.equal(names["w"], names["master"].bfloat16())
