"""4-bit key/value caches (d1_kv4_append, d1_kv4_load, d1_flash_attn_kv4, d1_kv4_mass, d1_kv4_evict) against plain
64-bit implementations of their definitions in include/d1kernels.h, written here in numpy.

Tolerances. Codes, parameters, read-back values, kept indices and moved rows are compared bit for bit. Of the attention:
  scores: fp16 products are exact in fp32; 64 of them are summed with at most one step of 2^-23 each (the tensor core may
    truncate), so a score is off by ds <= 2^-23 * 64 * scale * sum |q k|, plus a rounding of the scaled score
  weights: ex2 within 2^-13 (the coarsest form used, a cubic, is within 7.5e-5), one rounding to fp16 (2^-11 relative,
    2^-25 absolute below the normal range); the output one more rounding to fp16
  so |dO| <= (2^-11 + 2^-13 + 2 ds) sum p |v| + n 2^-25 max |v| + 2^-11 |O| + 2^-25, |d lse| <= ds + 2^-13 + 2^-21 |lse|
  mass: |d mass| <= sum over rows of w (ds + 2^-22 (2 + |s| + |lse|)) + rows * 2^-24 * mass; |s|, |lse| <= 32 here in
    log2 units, and the exponent's own rounding counts in them."""
import ctypes as C
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")
gpu = pytest.mark.gpu
INF = float("inf")


# ------------------------------------------------------------------------------------------------ plain forms
def quantise(x):
    """fp16 [..., 64] -> (codes, step, zero), by the definition in 64 bits."""
    x = np.asarray(x, np.float64)
    lo, hi = np.minimum(x.min(-1), 0), np.maximum(x.max(-1), 0)
    want = (hi - lo) / 15
    e = np.frexp(want)[1]
    unit = np.exp2(np.maximum(e - 7.0, -20.0))
    step = np.where(want > 0, np.ceil(want / unit) * unit, 0)
    s = np.where(step > 0, step, 1)
    zero = np.minimum(np.rint(-lo / s), 15)
    top = np.floor(65504 / s)[..., None]
    code = np.clip(np.clip(np.rint(x / s[..., None]), -top, top) + zero[..., None], 0, 15)
    return code.astype(np.int64), step, zero.astype(np.int64)


def pack(x):
    """fp16 [..., 64] -> (bytes [..., 32], parameters uint16 [...])."""
    code, step, zero = quantise(x)
    c = code.reshape(*code.shape[:-1], 8, 4, 2)
    word = sum((c[..., n, h] << (4 * n + 16 * h)) for n in range(4) for h in range(2)).astype(np.uint32)
    half = step.astype(np.float16)
    assert (half.astype(np.float64) == step).all() and (half.view(np.uint16) & 15 == 0).all()
    return word.view(np.uint8).reshape(*code.shape[:-1], 32), half.view(np.uint16) | zero.astype(np.uint16)


def values(b, par):
    w = np.ascontiguousarray(b).view(np.uint32)
    c = np.stack([(w >> (4 * n + 16 * h)) & 15 for n in range(4) for h in range(2)], -1)
    c = c.reshape(*b.shape[:-1], 64).astype(np.float64)
    step = (par & 0xFFF0).astype(np.uint16).view(np.float16).astype(np.float64)
    return (c - (par & 15)[..., None]) * step[..., None]


def keep_set(mass, keep, recent):
    """Kept indices of one head by the definition: the recent ones, and by (largest mass, lowest index)."""
    n = len(mass)
    keep = min(keep, n)
    recent = min(recent, keep)
    m = [-INF if math.isnan(v) else float(v) for v in mass[:n - recent]]
    best = sorted(range(n - recent), key=lambda i: (-m[i], i))[:keep - recent]
    return sorted(best) + list(range(n - recent, n))


# ------------------------------------------------------------------------------------------------ set-up
def vectors(rng, *shape):
    return (rng.standard_normal((*shape, 64)) * np.exp(0.5 * rng.standard_normal((*shape, 1)))).astype(np.float16)


class Caches:
    """Caches of the given lengths on the device: [cache][kv head][cap], rows behind a cache's last one poisoned."""

    def __init__(self, rng, lens, kvh, cap=None, empty=False):
        self.lens, self.kvh = lens, kvh
        self.cap = cap if cap is not None else max(8, -(-max(lens, default=0) // 8) * 8)
        n = len(lens)
        self.host = {"k4": np.full((n, kvh, self.cap, 32), 0xA5, np.uint8), "v4": np.full((n, kvh, self.cap, 32), 0xA5, np.uint8),
                     "kp": np.full((n, kvh, self.cap), 0x7E0F, np.uint16), "vp": np.full((n, kvh, self.cap), 0x7E0F, np.uint16)}
        for i, m in enumerate(lens):
            if m and not empty:
                self.host["k4"][i, :, :m], self.host["kp"][i, :, :m] = pack(vectors(rng, kvh, m))
                self.host["v4"][i, :, :m], self.host["vp"][i, :, :m] = pack(vectors(rng, kvh, m))
        self.dev = {k: torch.from_numpy(v.view(np.uint8) if v.dtype == np.uint8 else v.view(np.int16)).cuda()
                    for k, v in self.host.items()}
        self.mass = torch.full((n, kvh, self.cap), float("nan"), device="cuda")

    def fill(self, entry, i, mass=False):
        for k, v in self.dev.items():
            setattr(entry, k, v[i].data_ptr())
        if mass:
            entry.mass = self.mass[i].data_ptr()

    def values(self, i):
        m = self.lens[i]
        return [values(self.host[a][i, :, :m], self.host[p][i, :, :m]) for a, p in (("k4", "kp"), ("v4", "vp"))]

    def back(self):
        return {k: v.cpu().numpy().view(self.host[k].dtype) for k, v in self.dev.items()}


def table(pkg, seqs, caches=None, of=None, mass=False):
    """seqs: dicts of Kv4Seq fields. of[i]: the sequence's cache (None: none)."""
    arr = (pkg.abi.Kv4Seq * max(1, len(seqs)))()
    for i, s in enumerate(seqs):
        if caches is not None and of[i] is not None:
            caches.fill(arr[i], of[i], mass)
            arr[i].ext_len, arr[i].ext_cap = caches.lens[of[i]], caches.cap
        for k, v in s.items():
            setattr(arr[i], k, v)
    return torch.frombuffer(bytearray(bytes(arr)), dtype=torch.uint8).cuda()


def P(t):
    return t.data_ptr() if t is not None else None


def ST():
    return torch.cuda.current_stream().cuda_stream


def poisoned_rows(rng, spans, cols, gap=3):
    """Packed rows with `gap` NaN rows before and behind every span. -> (host rows, starts)"""
    starts, at = [], gap
    for n in spans:
        starts.append(at)
        at += n + gap
    x = np.full((at, cols), np.nan, np.float16)
    for s, n in zip(starts, spans):
        x[s:s + n] = rng.standard_normal((n, cols))
    return x, starts


# ------------------------------------------------------------------------------------------------ refusals (CPU)
def test_struct_layouts(pkg):
    a = pkg.abi
    assert C.sizeof(a.Kv4Seq) == 64 and a.Kv4Seq.k4.offset == 24 and a.Kv4Seq.mass.offset == 56
    assert C.sizeof(a.Kv4Evict) == 112 and a.Kv4Evict.k4.offset == 24 and a.Kv4Evict.kept.offset == 104


def test_plain_format():
    """The definition itself: at most half a step off, ranges covered, values exact in fp16."""
    rng = np.random.default_rng(0)
    x = np.concatenate([vectors(rng, 200), np.abs(vectors(rng, 50)), -np.abs(vectors(rng, 50)),
                        vectors(rng, 50) * np.float16(2.0 ** -16), np.zeros((1, 64), np.float16)])
    code, step, zero = quantise(x)
    v = values(*pack(x))
    assert (np.abs(v - x.astype(np.float64)) <= step[:, None] / 2).all()
    assert (v.astype(np.float16).astype(np.float64) == v).all()


def test_refusals(pkg):
    """Bad arguments are refused before anything is launched (no GPU needed); no work is a no-op."""
    lib, A, B = pkg.lib(), 1 << 20, 1 << 21  # never dereferenced
    att = lambda **k: lib.d1_flash_attn_kv4(*{**dict(Q=A, ldq=128, K=A, V=A, ldkv=64, O=A, ldo=128, lse=B, lse_ld=9, seqs=B,  # noqa: E731
        n=1, max_q=1, max_keys=1, heads=2, group=2, scale=0.125, q_rows=9, kv_rows=9, st=None), **k}.values())
    for bad in (dict(Q=None), dict(O=None), dict(seqs=None), dict(K=None), dict(V=None), dict(ldq=120), dict(ldo=64),
                dict(ldkv=56), dict(ldq=132), dict(Q=A + 8), dict(O=A + 2), dict(V=A + 4), dict(n=-1), dict(heads=0),
                dict(group=0), dict(heads=3), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(q_rows=-1),
                dict(kv_rows=-1), dict(lse_ld=8), dict(max_q=-1), dict(max_keys=-1), dict(heads=5000, group=1, ldq=320000, ldo=320000)):
        assert att(**bad) == -1, bad
    assert att(n=0) == 0 and att(q_rows=0) == 0
    app = lambda **k: lib.d1_kv4_append(*{**dict(K=A, V=A, ldkv=128, seqs=B, n=1, max_rows=1, kvh=2, st=None), **k}.values())  # noqa: E731
    load = lambda **k: lib.d1_kv4_load(*{**dict(seqs=B, n=1, max_rows=1, kvh=2, K=A, V=A, ldkv=128, st=None), **k}.values())  # noqa: E731
    for f in (app, load):
        for bad in (dict(K=None), dict(V=None), dict(seqs=None), dict(ldkv=64), dict(ldkv=132), dict(K=A + 8), dict(n=-2),
                    dict(kvh=0), dict(kvh=5000, ldkv=320000), dict(max_rows=-1)):
            assert f(**bad) == -1, bad
        assert f(n=0) == 0
    mass = lambda **k: lib.d1_kv4_mass(*{**dict(Q=A, ldq=128, lse=B, lse_ld=9, seqs=B, n=1, max_q=1, max_len=1, heads=2,  # noqa: E731
        group=2, scale=0.125, acc=0, q_rows=9, st=None), **k}.values())
    for bad in (dict(Q=None), dict(lse=None), dict(seqs=None), dict(ldq=64), dict(ldq=132), dict(Q=A + 8), dict(lse_ld=8),
                dict(n=-1), dict(heads=3), dict(group=0), dict(scale=0.0), dict(q_rows=-1), dict(max_q=-1), dict(max_len=-1)):
        assert mass(**bad) == -1, bad
    assert mass(n=0) == 0
    ev = lambda **k: lib.d1_kv4_evict(*{**dict(items=B, n=1, max_len=1, kvh=2, st=None), **k}.values())  # noqa: E731
    for bad in (dict(items=None), dict(n=-1), dict(kvh=0), dict(max_len=-1), dict(kvh=5000)):
        assert ev(**bad) == -1, bad
    assert ev(n=0) == 0


def test_refusals_of_alignment(pkg):
    """Tables off 8 bytes and log-sum-exps off 4 are refused before anything is launched."""
    lib, A = pkg.lib(), 1 << 20  # never dereferenced
    for at in (1, 2, 4):
        assert lib.d1_kv4_append(A, A, 128, A + at, 1, 1, 2, None) == -1
        assert lib.d1_kv4_load(A + at, 1, 1, 2, A, A, 128, None) == -1
        assert lib.d1_kv4_evict(A + at, 1, 1, 2, None) == -1
        for lse, seqs in ((A, A + at), (A + at % 4, A)):
            if lse == seqs:
                continue
            assert lib.d1_flash_attn_kv4(A, 128, A, A, 64, A, 128, lse, 9, seqs, 1, 1, 1, 2, 2, 0.125, 9, 9, None) == -1
            assert lib.d1_kv4_mass(A, 128, lse, 9, seqs, 1, 1, 1, 2, 2, 0.125, 0, 9, None) == -1


# ------------------------------------------------------------------------------------------------ append, load
def special_vectors():
    """Vectors at the format's borders."""
    rng = np.random.default_rng(5)
    x = [np.zeros(64), np.full(64, 3.25), np.full(64, -0.1), np.linspace(-65504, 65504, 64), np.linspace(0, 65504, 64),
         np.linspace(-65504, 0, 64), np.full(64, 2.0 ** -24), rng.standard_normal(64) * 2.0 ** -18,
         rng.standard_normal(64) * 2.0 ** -12, np.where(np.arange(64) == 7, 1000.0, 2.0 ** -10),
         np.tile([-7.5, 7.5], 32), np.tile(np.arange(-8, 8) + 0.5, 4), np.tile(np.arange(16) - 7.0, 4),
         np.tile(np.arange(0, 15.5, 0.5), 3)[:64]]
    for s in (1.0, 0.25, 96.0, 2.0 ** -9):  # many quotients that end in exactly one half
        x += [np.clip((np.arange(64) % 31 - 15) * 0.5 * s, -7.5 * s, 7.5 * s)]
    return np.asarray(x).astype(np.float16)


@gpu
@pytest.mark.parametrize("rows,ext,kvh", [([1], [0], 1), ([1, 1, 1], [0, 7, 1023], 8), ([5, 0, 130, 33], [3, 9, 0, 64], 3),
                                          ([257], [1], 16)])
def test_append_load(pkg, gpu_lib, rows, ext, kvh):
    rng = np.random.default_rng(sum(rows) + kvh)
    cap = -(-max(a + b for a, b in zip(rows, ext)) // 8) * 8 + 8
    c = Caches(rng, ext, kvh, cap)
    x, starts = poisoned_rows(rng, rows, 3 * kvh * 64 + 8)
    d = torch.from_numpy(x).cuda()
    tab = table(pkg, [dict(kv_start=s, kv_len=n) for s, n in zip(starts, rows)], c, range(len(rows)))
    ld, ko, vo = x.shape[1], kvh * 64, 2 * kvh * 64
    assert gpu_lib.d1_kv4_append(d[:, ko:].data_ptr(), d[:, vo:].data_ptr(), ld, P(tab), len(rows), max(rows), kvh, ST()) == 0
    got = c.back()
    want = {k: v.copy() for k, v in c.host.items()}
    for i, (s, n, e) in enumerate(zip(starts, rows, ext)):
        for a, p, o in (("k4", "kp", ko), ("v4", "vp", vo)):
            b, par = pack(x[s:s + n, o:o + kvh * 64].reshape(n, kvh, 64).transpose(1, 0, 2)) if n else (0, 0)
            if n:
                want[a][i, :, e:e + n], want[p][i, :, e:e + n] = b, par
    for k in want:
        assert (got[k] == want[k]).all(), k
    # back again, into rows with other contents around them
    y = torch.full((x.shape[0], 2 * kvh * 64), 7.0, dtype=torch.float16, device="cuda")
    assert gpu_lib.d1_kv4_load(P(tab), len(rows), 1, kvh, P(y), y[:, kvh * 64:].data_ptr(), 2 * kvh * 64, ST()) == 0
    assert gpu_lib.d1_kv4_error() == 0
    ref = np.full(y.shape, 7.0)
    for i, (s, n, e) in enumerate(zip(starts, rows, ext)):
        for j, (a, p) in enumerate((("k4", "kp"), ("v4", "vp"))):
            v = values(want[a][i, :, e:e + n], want[p][i, :, e:e + n])
            ref[s:s + n, j * kvh * 64:(j + 1) * kvh * 64] = v.transpose(1, 0, 2).reshape(n, kvh * 64)
    assert (y.double().cpu().numpy() == ref).all()


@gpu
def test_append_borders(pkg, gpu_lib):
    """Ranges on one side of zero, the largest and smallest numbers, exact halves; NaN and infinities read as NaN."""
    x = special_vectors()
    n = len(x)
    bad = np.zeros((4, 64), np.float16)
    bad[0, 3], bad[1, 60], bad[2, 0], bad[3] = np.nan, np.inf, -np.inf, np.nan
    rng = np.random.default_rng(0)
    c = Caches(rng, [0], 1, 64)
    d = torch.from_numpy(np.concatenate([x, bad])).cuda()
    tab = table(pkg, [dict(kv_start=0, kv_len=n + 4)], c, [0])
    assert gpu_lib.d1_kv4_append(P(d), P(d), 64, P(tab), 1, n + 4, 1, ST()) == 0
    got = c.back()
    b, par = pack(x)
    assert (got["kp"][0, 0, :n] == par).all() and (got["k4"][0, 0, :n] == b).all()
    assert (got["vp"][0, 0, :n] == par).all() and (got["v4"][0, 0, :n] == b).all()
    y = torch.zeros(n + 4, 128, dtype=torch.float16, device="cuda")
    assert gpu_lib.d1_kv4_load(P(tab), 1, n + 4, 1, P(y), y[:, 64:].data_ptr(), 128, ST()) == 0
    y = y.double().cpu().numpy()
    assert np.isfinite(y[:n]).all() and np.isnan(y[n:]).all()
    assert gpu_lib.d1_kv4_error() == 0


# ------------------------------------------------------------------------------------------------ attention
def plain_attend(x, seqs, caches, of, kvh, group, scale, own):
    """64-bit attention -> O, lse, and the tolerances of both (see the top)."""
    h = kvh * group
    O, L = np.full((x.shape[0], h * 64), np.nan), np.full((h, x.shape[0]), np.nan)
    tO, tL = np.zeros_like(O), np.zeros_like(L)
    x = x.astype(np.float64)
    for i, s in enumerate(seqs):
        ck, cv = caches.values(of[i]) if of[i] is not None else (np.zeros((kvh, 0, 64)),) * 2
        r, kv = slice(s["q_start"], s["q_start"] + s["q_len"]), slice(s["kv_start"], s["kv_start"] + s["kv_len"])
        for j in range(h):
            g = j // group
            q = x[r, j * 64:(j + 1) * 64]
            K = np.concatenate([ck[g], x[kv, (h + g) * 64:(h + g + 1) * 64]])
            V = np.concatenate([cv[g], x[kv, (h + kvh + g) * 64:(h + kvh + g + 1) * 64]])
            if not len(K):
                O[r, j * 64:(j + 1) * 64], L[j, r] = 0, -INF
                continue
            y = q @ K.T * scale
            m = y.max(-1, keepdims=True, initial=-INF)
            p = np.exp(y - m)
            l = p.sum(-1, keepdims=True)
            p /= l
            o = p @ V
            ds = 2.0 ** -23 * (64 * scale * (np.abs(q) @ np.abs(K).T).max(-1, keepdims=True) + np.abs(m) + 1)
            O[r, j * 64:(j + 1) * 64], L[j, r] = o, (m + np.log(l))[:, 0]
            tO[r, j * 64:(j + 1) * 64] = ((2.0 ** -11 + 2.0 ** -13 + 2 * ds) * (p @ np.abs(V)) +
                                          len(K) * 2.0 ** -25 * np.abs(V).max() + 2.0 ** -11 * np.abs(o) + 2.0 ** -25)
            tL[j, r] = (ds + 2.0 ** -13)[:, 0] + 2.0 ** -21 * np.abs(L[j, r])
    return O, L, tO, tL


def attend(gpu_lib, x, tab, n, kvh, group, scale=0.125, max_q=None, max_keys=0, ld_o=None, lse=True):
    h, rows = kvh * group, x.shape[0]
    d = x if torch.is_tensor(x) else torch.from_numpy(x).cuda()
    ldo = ld_o or h * 64
    O = torch.full((rows, ldo), 7.0, dtype=torch.float16, device="cuda")
    L = torch.full((h, rows + 5), 7.0, device="cuda") if lse else None
    r = gpu_lib.d1_flash_attn_kv4(P(d), d.shape[1], d[:, h * 64:].data_ptr(), d[:, (h + kvh) * 64:].data_ptr(), d.shape[1],
                                  P(O), ldo, P(L), rows + 5, P(tab), n, max_q, max_keys, h, group, scale, rows, rows, ST())
    assert r == 0
    torch.cuda.synchronize()
    return O, L


def check_attend(O, L, want, h):
    o, l, tO, tL = want
    got, none = O.double().cpu().numpy(), np.isnan(o[:, 0])
    assert (got[none] == 7).all() and (got[:, h * 64:] == 7).all()  # rows and columns that belong to nobody
    assert (np.abs(got[~none, :h * 64] - o[~none]) <= tO[~none]).all(), np.nanmax(np.abs(got[:, :h * 64] - o) / tO)
    if L is not None:
        got = L.double().cpu().numpy()
        assert (got[:, len(o):] == 7).all() and (got[:, :len(o)][:, none] == 7).all()
        got, l, tL = got[:, :len(o)][:, ~none], l[:, ~none], tL[:, ~none]
        fin = np.isfinite(l)
        assert (got[~fin] == l[~fin]).all() and (np.abs(got[fin] - l[fin]) <= tL[fin]).all()


# which kernel runs, and whether a cluster of CTAs shares a unit, follows from max_q; the results must not
HINTS = [1, 17, 40, 200, 5000]
CASES = {
    "one": ([1], [1], [0], 8, 2),
    "no keys": ([3, 1, 200], [0, 5, 0], [0, 0, 0], 4, 2),
    "own rows only": ([65, 1], [0, 0], [65, 1], 2, 2),
    "tile edges": ([1, 7, 8, 9], [63, 64, 65, 128], [0, 0, 1, 64], 2, 2),
    "large tile edges": ([127, 128, 129, 255, 257], [127, 128, 129, 256, 1], [128, 127, 1, 129, 257], 1, 2),
    "odd": ([33, 1, 0, 300], [517, 1000, 33, 3], [33, 1, 0, 300], 3, 3),
    "one head each": ([5, 131], [700, 129], [5, 131], 3, 1),
    "wide groups": ([2, 40], [300, 777], [2, 40], 2, 8),
    "group of five": ([19, 150], [400, 130], [0, 150], 1, 5),
    "long": ([3, 2], [16384, 5003], [3, 2], 1, 2),
    "many sequences": ([1 + i % 5 for i in range(300)], [i % 140 for i in range(300)], [i % 3 for i in range(300)], 1, 2),
    "two runs of units": ([130 if i % 7 == 0 else 1 for i in range(260)], [i % 9 for i in range(260)], [0] * 260, 1, 2),
}


@gpu
@pytest.mark.parametrize("max_q", HINTS)
@pytest.mark.parametrize("name", CASES)
def test_attend(pkg, gpu_lib, name, max_q):
    q, ext, kv, kvh, group = CASES[name]
    rng = np.random.default_rng(len(name))
    h = kvh * group
    c = Caches(rng, ext, kvh, -(-max(ext) // 8) * 8 + 16)
    x, starts = poisoned_rows(rng, [max(a, b) for a, b in zip(q, kv)], (h + 2 * kvh) * 64 + 16)
    seqs = [dict(q_start=s, q_len=a, kv_start=s, kv_len=b) for s, a, b in zip(starts, q, kv)]
    tab = table(pkg, seqs, c, range(len(q)))
    O, L = attend(gpu_lib, x, tab, len(q), kvh, group, max_q=max_q, max_keys=max(ext), ld_o=h * 64 + 24)
    assert gpu_lib.d1_kv4_error() == 0
    check_attend(O, L, plain_attend(x, seqs, c, list(range(len(q))), kvh, group, 0.125, True), h)


@gpu
@pytest.mark.parametrize("max_q", HINTS)
def test_attend_sharp_and_shared(pkg, gpu_lib, max_q):
    """Large scores (one key takes nearly all), a cache that several sequences share, no lse, another scale."""
    rng = np.random.default_rng(3)
    kvh, group, of = 2, 2, [0, 1, 0, None, 0]
    c = Caches(rng, [333, 40], kvh)
    q = [40, 3, 130, 9, 1]
    x, starts = poisoned_rows(rng, q, (kvh * group + 2 * kvh) * 64)
    seqs = [dict(q_start=s, q_len=a, kv_start=s, kv_len=a) for s, a in zip(starts, q)]
    tab = table(pkg, seqs, c, of)
    for scale in (0.125, 2.0):
        O, _ = attend(gpu_lib, x, tab, 5, kvh, group, scale, max_q, 400, lse=False)
        check_attend(O, None, plain_attend(x, seqs, c, of, kvh, group, scale, True), kvh * group)
    assert gpu_lib.d1_kv4_error() == 0


SHARED_OUT = {
    "packed": ([30, 1, 0, 50], [1300, 0, 128, 257], [30, 0, 0, 1], 2, 2),
    "pairs": ([200, 129], [700, 5], [50, 0], 1, 2),
    "single": ([300, 20], [257, 640], [0, 20], 1, 1),
    "three heads": ([50, 90, 3], [1000, 3, 129], [0, 90, 0], 1, 3),
    "long": ([64], [9000], [64], 2, 2),
}


@gpu
@pytest.mark.parametrize("max_keys", [1300, 3500, 40000])
@pytest.mark.parametrize("max_q", [1, 12, 70, 128])
@pytest.mark.parametrize("name", SHARED_OUT)
def test_attend_shared_out(pkg, gpu_lib, name, max_q, max_keys):
    """Clusters of CTAs share out the keys, be there fewer than CTAs, none, or more units than clusters; a bad entry among
    the others is skipped. The same call gives the same bits."""
    q, ext, kv, kvh, group = SHARED_OUT[name]
    rng = np.random.default_rng(len(name) + 40)
    h = kvh * group
    c = Caches(rng, ext, kvh, -(-max(ext) // 8) * 8)
    x, starts = poisoned_rows(rng, [max(a, b) for a, b in zip(q, kv)], (h + 2 * kvh) * 64)
    seqs = [dict(q_start=s, q_len=a, kv_start=s, kv_len=b) for s, a, b in zip(starts, q, kv)]
    want = plain_attend(x, seqs, c, list(range(len(q))), kvh, group, 0.125, True)
    first = None
    for bad in ([], [dict(q_start=0, q_len=5, kv_start=-1, kv_len=7)]):
        for _ in range(2):
            O, L = attend(gpu_lib, x, table(pkg, bad + seqs, c, [None] * len(bad) + list(range(len(q)))), len(bad + seqs), kvh,
                          group, 0.125, max_q, max_keys)
            assert (gpu_lib.d1_kv4_error() != 0) == bool(bad)
            check_attend(O, L, want, h)
            if not bad:
                assert first is None or torch.equal(O, first)
                first = O


@gpu
@pytest.mark.parametrize("max_q", HINTS)
def test_lse_of_few_keys(pkg, gpu_lib, max_q):
    """Single exponentials are not averaged out: beside the scores' own error (ds) 2^-22 of an exponential, at most 24 rounded
    additions and rescalings (2^-19.4) and the logarithm's and its factor's roundings, 2^-21 of the result."""
    rng = np.random.default_rng(13)
    kvh, group, q, ext = 2, 2, [130, 40, 70, 3, 200], [2, 16, 31, 128, 9]
    h = kvh * group
    c = Caches(rng, ext, kvh, 136)
    x, starts = poisoned_rows(rng, q, (h + 2 * kvh) * 64)
    seqs = [dict(q_start=s, q_len=a, kv_start=s, kv_len=0) for s, a in zip(starts, q)]
    _, L = attend(gpu_lib, x, table(pkg, seqs, c, range(5)), 5, kvh, group, 0.125, max_q, 128)
    _, l, _, tL = plain_attend(x, seqs, c, range(5), kvh, group, 0.125, True)
    ok = np.isfinite(l)
    tight = tL - 2.0 ** -13 + 2.0 ** -22 + 2.0 ** -19.4
    assert (np.abs(L.double().cpu().numpy()[:, :len(x)] - l)[ok] <= tight[ok]).all()


@gpu
@pytest.mark.parametrize("at", [0, 15, 50, 78, 99])
@pytest.mark.parametrize("max_q", HINTS)
def test_attend_nan_stays_in_its_rows(pkg, gpu_lib, max_q, at):
    """A NaN key makes its sequence's rows NaN, a NaN query row only itself, as in fp16; other sequences keep theirs."""
    rng = np.random.default_rng(4)
    kvh, group = 2, 2
    c = Caches(rng, [100, 100], kvh)
    c.dev["kp"][0, 1, at] = 0x7E00
    x, starts = poisoned_rows(rng, [4, 4], (kvh * group + 2 * kvh) * 64)
    x[starts[1] + 2, :64] = np.nan
    seqs = [dict(q_start=s, q_len=4, kv_start=s, kv_len=0) for s in starts]
    O, L = attend(gpu_lib, x, table(pkg, seqs, c, [0, 1]), 2, kvh, group, 0.125, max_q, 100)
    o = O.float().cpu().numpy().reshape(len(x), 4, 64)
    nan = np.isnan(o).any(-1)
    want = np.zeros_like(nan)
    want[starts[0]:starts[0] + 4, 2:] = True  # heads of kv head 1
    want[starts[1] + 2, 0] = True
    assert (nan == want).all() and (np.isnan(L.cpu().numpy()[:, :len(x)].T) == want).all()


# ------------------------------------------------------------------------------------------------ mass
def plain_mass(x, lse, seqs, caches, of, kvh, group, scale):
    n = len(caches.lens)
    M, T = np.zeros((n, kvh, caches.cap)), np.zeros((n, kvh, caches.cap))
    x, rows = x.astype(np.float64), np.zeros(n)
    for i, s in enumerate(seqs):
        r, e = slice(s["q_start"], s["q_start"] + s["q_len"]), caches.lens[of[i]]
        K = caches.values(of[i])[0]
        rows[of[i]] += s["q_len"] * group
        for j in range(kvh * group):
            q, k = x[r, j * 64:(j + 1) * 64], K[j // group]
            y = q @ k.T * scale
            l = lse[j, r].astype(np.float64)[:, None]
            w = np.where(l > -INF, np.exp(y - l), 0)
            ds = 2.0 ** -23 * 64 * scale * (np.abs(q) @ np.abs(k).T) + 2.0 ** -22 * (2 + 1.5 * np.abs(y) + 1.5 * np.abs(np.where(l > -INF, l, 0)))
            M[of[i], j // group, :e] += w.sum(0)
            T[of[i], j // group, :e] += (w * ds).sum(0)
    return M, T + rows[:, None, None] * 2.0 ** -24 * M + 1e-30


MASSES = {
    "one": ([1], [1], [0], 8, 2),
    "edges": ([1, 7, 8, 9, 16], [63, 64, 65, 128, 513], [0, 1, 2, 3, 4], 2, 2),
    "large edges": ([127, 256, 257, 600], [127, 128, 129, 700], [0, 1, 2, 3], 1, 2),
    "shared": ([30, 1, 0, 130, 5, 64], [1000, 77], [0, 1, 0, 0, 1, 0], 3, 3),
    "one head each": ([70, 9], [300, 12], [0, 1], 4, 1),
    "wide groups": ([40, 3], [300, 777], [0, 1], 2, 8),
    "many": ([2] * 300, [90], [0] * 300, 1, 2),
    "as many as a table holds": ([33] * 256, [130, 1, 260], [i % 3 for i in range(256)], 1, 2),
}


@gpu
@pytest.mark.parametrize("max_q", HINTS)
@pytest.mark.parametrize("name", MASSES)
def test_mass(pkg, gpu_lib, name, max_q):
    q, ext, of, kvh, group = MASSES[name]
    rng = np.random.default_rng(len(name))
    h = kvh * group
    c = Caches(rng, ext, kvh, -(-max(ext) // 8) * 8 + 8)
    x, starts = poisoned_rows(rng, q, h * 64 + 8)
    lse = (2 + rng.standard_normal((h, x.shape[0] + 3))).astype(np.float32)
    for i, s in enumerate(starts):  # rows without keys add nothing
        if q[i] > 2:
            lse[0, s + 1] = -INF
    seqs = [dict(q_start=s, q_len=a) for s, a in zip(starts, q)]
    tab = table(pkg, seqs, c, of, mass=True)
    d, l = torch.from_numpy(x).cuda(), torch.from_numpy(lse).cuda()
    call = lambda acc: gpu_lib.d1_kv4_mass(P(d), d.shape[1], P(l), lse.shape[1], P(tab), len(q), max_q, max(ext), h, group,  # noqa: E731
                                           0.125, acc, x.shape[0], ST())
    assert call(0) == 0
    M, T = plain_mass(x, lse, seqs, c, of, kvh, group, 0.125)
    got = c.mass.double().cpu().numpy()
    for i, e in enumerate(ext):
        assert np.isnan(got[i, :, e:]).all()
        assert (np.abs(got[i, :, :e] - M[i, :, :e]) <= T[i, :, :e]).all(), np.max(np.abs(got - M)[i, :, :e] / T[i, :, :e])
    once = c.mass.clone()
    assert call(1) == 0  # adds the same sums, bit for bit
    for i, e in enumerate(ext):
        assert torch.equal(c.mass[i, :, :e], once[i, :, :e] * 2)
    assert gpu_lib.d1_kv4_error() == 0


@gpu
@pytest.mark.parametrize("max_len", [0, 1, 300, 40000])
@pytest.mark.parametrize("max_q", HINTS)
def test_mass_wrong_hints(pkg, gpu_lib, max_q, max_len):
    """Rows and keys beyond the lengths given are computed all the same, however the CTAs are grouped."""
    rng = np.random.default_rng(14)
    kvh, group, q, ext, of = 2, 2, [300, 1, 700, 90], [700, 131, 1], [0, 1, 0, 2]
    h = kvh * group
    c = Caches(rng, ext, kvh, 704)
    x, starts = poisoned_rows(rng, q, h * 64)
    lse = (2 + rng.standard_normal((h, len(x)))).astype(np.float32)
    seqs = [dict(q_start=s, q_len=a) for s, a in zip(starts, q)]
    tab = table(pkg, seqs, c, of, mass=True)
    d, l = torch.from_numpy(x).cuda(), torch.from_numpy(lse).cuda()
    M, T = plain_mass(x, lse, seqs, c, of, kvh, group, 0.125)
    first = None
    for _ in range(3):
        c.mass.fill_(5)
        assert gpu_lib.d1_kv4_mass(P(d), d.shape[1], P(l), len(x), P(tab), len(q), max_q, max_len, h, group, 0.125, 0, len(x),
                                   ST()) == 0
        got = c.mass.double().cpu().numpy()
        for i, e in enumerate(ext):
            assert (got[i, :, e:] == 5).all() and (np.abs(got[i, :, :e] - M[i, :, :e]) <= T[i, :, :e]).all()
        assert first is None or (got == first).all()  # the same call, the same bits
        first = got
    assert gpu_lib.d1_kv4_error() == 0


@gpu
@pytest.mark.parametrize("max_q", HINTS)
def test_mass_of_rows_that_add_nothing(pkg, gpu_lib, max_q):
    """No rows: the sum is 0, and is written. Rows with lse = -inf add nothing, be they NaN (padding): the same bits as
    without them."""
    rng = np.random.default_rng(12)
    kvh, group, q, ext, of = 2, 2, [0, 70, 5, 0, 0, 64], [130, 77, 9], [0, 1, 1, 2, 2, 1]
    h = kvh * group
    c = Caches(rng, ext, kvh, 136)
    x, starts = poisoned_rows(rng, q, h * 64)
    lse = (2 + rng.standard_normal((h, len(x)))).astype(np.float32)
    seqs = [dict(q_start=s, q_len=a) for s, a in zip(starts, q)]
    tab = table(pkg, seqs, c, of, mass=True)
    pad = [starts[1], starts[1] + 40, starts[1] + 69, starts[2] + 4, starts[5] + 13]
    lse[:, pad] = -INF
    got = []
    for v in (0.5, np.nan, np.inf):
        x[pad] = v
        d, l = torch.from_numpy(x).cuda(), torch.from_numpy(lse).cuda()
        for acc in (0, 1):
            c.mass.fill_(3)
            assert gpu_lib.d1_kv4_mass(P(d), d.shape[1], P(l), len(x), P(tab), len(q), max_q, 130, h, group, 0.125, acc,
                                       len(x), ST()) == 0
            assert (c.mass[0, :, :130] == 3 * acc).all() and (c.mass[2, :, :9] == 3 * acc).all()
            assert all((c.mass[i, :, e:] == 3).all() for i, e in enumerate(ext))
        got.append(c.mass[1].clone())
    assert not torch.isnan(got[0]).any() and torch.equal(got[0], got[1]) and torch.equal(got[0], got[2])
    assert gpu_lib.d1_kv4_error() == 0


@gpu
def test_more_sequences_than_a_grid(pkg, gpu_lib):
    """Beyond 65535 sequences a CTA takes one after the other: long sums first, then short ones."""
    rng = np.random.default_rng(15)
    kvh, group, n = 1, 2, 65535 + 24
    h, at = kvh * group, list(range(24)) + list(range(65535, n))
    q = [61 - i % 7 if i < 24 else 1 + i % 9 for i in range(48)]
    c = Caches(rng, [30 + i for i in range(48)], kvh, 80)
    x, starts = poisoned_rows(rng, q, (h + 2 * kvh) * 64)
    lse = (2 + rng.standard_normal((h, len(x)))).astype(np.float32)
    seqs = [dict(q_start=s, q_len=m, kv_start=0, kv_len=0) for s, m in zip(starts, q)]
    some = bytes(table(pkg, seqs, c, range(48), mass=True).cpu().numpy())
    tab = bytearray(64 * n)
    for i, j in enumerate(at):
        tab[64 * j:64 * j + 64] = some[64 * i:64 * i + 64]
    tab = torch.frombuffer(tab, dtype=torch.uint8).cuda()
    d, l = torch.from_numpy(x).cuda(), torch.from_numpy(lse).cuda()
    M, T = plain_mass(x, lse, seqs, c, range(48), kvh, group, 0.125)
    want = plain_attend(x, seqs, c, range(48), kvh, group, 0.125, True)
    for _ in range(3):
        c.mass.fill_(5)
        assert gpu_lib.d1_kv4_mass(P(d), d.shape[1], P(l), len(x), P(tab), n, max(q), 80, h, group, 0.125, 0, len(x), ST()) == 0
        got = c.mass.double().cpu().numpy()
        for i, e in enumerate(c.lens):
            assert (got[i, :, e:] == 5).all() and (np.abs(got[i, :, :e] - M[i, :, :e]) <= T[i, :, :e]).all()
    for max_q in (1, 30, 61):
        O, L = attend(gpu_lib, d, tab, n, kvh, group, 0.125, max_q, 80)
        check_attend(O, L, want, h)
    assert gpu_lib.d1_kv4_error() == 0


@gpu
@pytest.mark.parametrize("max_q", [1, 64])
def test_mass_of_a_foreign_lse(pkg, gpu_lib, max_q):
    """An lse far from the scores, in each column of a piece of 32: e^80 is a number, e^95 is infinite, NaN stays, e^-120 and
    lse = inf add nothing. Scores are 0 here, and the 63 other columns add 1 each: a sum is off by at most 2^-22 of an
    exponential, 80 * 2^-23 of its exponent and 64 additions."""
    rng = np.random.default_rng(16)
    c = Caches(rng, [130], 1, 136)
    d = torch.zeros(32, 128, dtype=torch.float16, device="cuda")
    tab = table(pkg, [dict(q_start=0, q_len=32)], c, [0], mass=True)
    for at in range(32):
        for v, want in ((-80.0, math.exp(80)), (-95.0, INF), (-1e9, INF), (-1e30, INF), (120.0, 63.0), (INF, 63.0), (-INF, 63.0),
                        (np.nan, np.nan)):
            lse = torch.zeros(2, 32, device="cuda")
            lse[at % 2, at // 2] = v
            assert gpu_lib.d1_kv4_mass(P(d), 128, P(lse), 32, P(tab), 1, max_q, 130, 2, 2, 0.125, 0, 32, ST()) == 0
            got = c.mass[0, 0, :130].double().cpu().numpy()
            if math.isfinite(want):
                assert (np.abs(got - want) <= (2.0 ** -22 + 80 * 2.0 ** -23 + 64 * 2.0 ** -24) * want).all(), (at, v, got[0])
            else:
                assert np.array_equal(got, np.full(130, want), equal_nan=True), (at, v, got[0])
    assert gpu_lib.d1_kv4_error() == 0


# ------------------------------------------------------------------------------------------------ evict
@gpu
@pytest.mark.parametrize("lens,keep,recent,kvh", [([1], [1], [0], 1), ([9, 0, 100], [3, 5, 0], [0, 1, 4], 2),
                                                  ([1500, 700, 64], [750, 800, 64], [33, 5, 64], 8),
                                                  ([5000, 4099], [4097, 7], [9, 20], 3), ([16384], [4096], [64], 2),
                                                  ([40001], [20000], [1], 1)])
def test_evict(pkg, gpu_lib, lens, keep, recent, kvh):
    rng = np.random.default_rng(sum(lens))
    c = Caches(rng, lens, kvh)
    mass = np.floor(rng.random((len(lens), kvh, c.cap)) ** 4 * 50).astype(np.float32) / 8  # many equal ones
    mass[rng.random(mass.shape) < 0.02] = np.nan
    mass[rng.random(mass.shape) < 0.02] = -0.0
    mass[rng.random(mass.shape) < 0.01] = np.inf
    mass[rng.random(mass.shape) < 0.01] = -np.inf
    mass[rng.random(mass.shape) < 0.01] = -1.5
    md = torch.from_numpy(mass).cuda()
    d = Caches(rng, [0] * len(lens), kvh, max(8, -(-max(min(a, b) for a, b in zip(lens, keep)) // 8) * 8) + 8)
    kept = torch.full((len(lens), kvh, d.cap), -9, dtype=torch.int32, device="cuda")
    arr = (pkg.abi.Kv4Evict * len(lens))()
    for i in range(len(lens)):
        e = arr[i]
        e.len, e.cap, e.keep, e.recent, e.dst_cap, e.mass = lens[i], c.cap, keep[i], recent[i], d.cap, md[i].data_ptr()
        for k in c.dev:
            setattr(e, k, c.dev[k][i].data_ptr())
            setattr(e, "dst_" + k, d.dev[k][i].data_ptr())
        e.dst_mass = d.mass[i].data_ptr() if i != 1 else None
        e.kept = kept[i].data_ptr() if i != 2 else None
    items = torch.frombuffer(bytearray(bytes(arr)), dtype=torch.uint8).cuda()
    assert gpu_lib.d1_kv4_evict(P(items), len(lens), max(lens), kvh, ST()) == 0
    assert gpu_lib.d1_kv4_error() == 0
    got, got_m, got_k = d.back(), d.mass.cpu().numpy(), kept.cpu().numpy()
    for i, n in enumerate(lens):
        for g in range(kvh):
            at = keep_set(mass[i, g, :n], keep[i], recent[i])
            m = len(at)
            assert (got_k[i, g, :m] == (at if i != 2 else -9)).all() and (got_k[i, g, m:] == -9).all()
            for k in got:
                assert (got[k][i, g, :m] == c.host[k][i, g, at]).all() and (got[k][i, g, m:] == d.host[k][i, g, m:]).all()
            if i != 1:
                assert np.array_equal(got_m[i, g, :m], mass[i, g, at], equal_nan=True)
            assert np.isnan(got_m[i, g, m if i != 1 else 0:]).all()


# ------------------------------------------------------------------------------------------------ tables
@gpu
@pytest.mark.parametrize("max_q", HINTS)
def test_bad_entries_are_skipped(pkg, gpu_lib, max_q):
    """Entries that break the table's rules are skipped and reported; the others are computed. All of these are refused by
    the kernels' own checks before any access."""
    rng = np.random.default_rng(6)
    kvh, group, n = 2, 2, 4
    h = kvh * group
    c = Caches(rng, [40] * n, kvh, 56)
    x, starts = poisoned_rows(rng, [9] * n, (h + 2 * kvh) * 64)
    rows = len(x)
    good = [dict(q_start=s, q_len=9, kv_start=s, kv_len=9) for s in starts]
    d = torch.from_numpy(x).cuda()
    lse = torch.full((h, rows), 3.0, device="cuda")
    for bad in (dict(ext_len=57), dict(ext_len=-1), dict(ext_cap=52), dict(k4=None), dict(vp=None),
                dict(v4=c.dev["v4"].data_ptr() + 8), dict(kp=c.dev["kp"].data_ptr() + 2), dict(q_len=rows), dict(q_start=-1),
                dict(q_len=-1), dict(q_start=2 ** 31 - 1), dict(ext_cap=2 ** 30 + 8)):
        for at in (0, 2):
            seqs = [dict(s) for s in good]
            seqs[at].update(bad)
            tab = table(pkg, seqs, c, range(n), mass=True)
            O, L = attend(gpu_lib, d, tab, n, kvh, group, 0.125, max_q, 60)
            assert gpu_lib.d1_kv4_error() != 0 and gpu_lib.d1_kv4_error() == 0
            keep = [i for i in range(n) if i != at]
            want = plain_attend(x, [good[i] for i in keep], c, keep, kvh, group, 0.125, True)
            check_attend(O, L, want, h)
            c.mass.fill_(7)
            assert gpu_lib.d1_kv4_mass(P(d), d.shape[1], P(lse), rows, P(tab), n, max_q, 40, h, group, 0.125, 0, rows, ST()) == 0
            assert gpu_lib.d1_kv4_error() != 0
            assert (c.mass[at] == 7).all() and all((c.mass[i, :, :40] != 7).all() for i in keep)
    for bad in (dict(kv_len=17), dict(kv_len=-1), dict(kv_start=-1), dict(ext_len=57), dict(ext_cap=52), dict(kp=None)):
        seqs = [dict(s) for s in good]
        seqs[1].update(bad)
        tab = table(pkg, seqs, c, range(n))
        before = c.back()
        assert gpu_lib.d1_kv4_append(P(d), P(d), d.shape[1], P(tab), n, 9, kvh, ST()) == 0
        assert gpu_lib.d1_kv4_error() != 0
        after = c.back()
        assert all((after[k][1] == before[k][1]).all() for k in after)
        assert all((after["kp"][i, :, 40:49] != 0x7E0F).all() for i in (0, 2, 3))


@gpu
@pytest.mark.parametrize("max_q", HINTS)
def test_bad_entries_of_a_shared_mass(pkg, gpu_lib, max_q):
    """An entry that is skipped takes none of those with it that share its mass array, be it before or behind them."""
    rng = np.random.default_rng(17)
    kvh, group, q = 2, 2, [9, 70, 33, 5]
    h = kvh * group
    c = Caches(rng, [140, 40], kvh, 144)
    x, starts = poisoned_rows(rng, q, h * 64)
    lse = (2 + rng.standard_normal((h, len(x)))).astype(np.float32)
    d, l = torch.from_numpy(x).cuda(), torch.from_numpy(lse).cuda()
    good, of = [dict(q_start=s, q_len=m) for s, m in zip(starts, q)], [0, 0, 1, 0]
    for at in (0, 1, 3):
        keep = [i for i in range(4) if i != at]
        M, T = plain_mass(x, lse, [good[i] for i in keep], c, [of[i] for i in keep], kvh, group, 0.125)
        for bad in (dict(ext_len=145), dict(k4=None), dict(ext_cap=140), dict(q_len=len(x) + 1), dict(kp=c.dev["kp"].data_ptr() + 2)):
            seqs = [dict(s) for s in good]
            seqs[at].update(bad)
            c.mass.fill_(7)
            assert gpu_lib.d1_kv4_mass(P(d), d.shape[1], P(l), len(x), P(table(pkg, seqs, c, of, mass=True)), 4, max_q, 140, h, group,
                                       0.125, 0, len(x), ST()) == 0
            assert gpu_lib.d1_kv4_error() != 0
            got = c.mass.double().cpu().numpy()
            for i, e in enumerate((140, 40)):
                assert (got[i, :, e:] == 7).all() and (np.abs(got[i, :, :e] - M[i, :, :e]) <= T[i, :, :e]).all(), (at, bad, i)


@gpu
@pytest.mark.parametrize("off", [1, 2, 3])
def test_masses_off_four_bytes_are_refused(pkg, gpu_lib, off):
    """mass, dst_mass and kept off 4 bytes: the entry is skipped and reported, the others are computed."""
    rng = np.random.default_rng(18)
    c, d = Caches(rng, [140, 40], 2, 144), Caches(rng, [0, 0], 2, 24)
    x, starts = poisoned_rows(rng, [9, 70], 4 * 64)
    lse = (2 + rng.standard_normal((4, len(x)))).astype(np.float32)
    dx, l = torch.from_numpy(x).cuda(), torch.from_numpy(lse).cuda()
    seqs = [dict(q_start=s, q_len=m) for s, m in zip(starts, (9, 70))]
    M, T = plain_mass(x, lse, seqs, c, [0, 1], 2, 2, 0.125)
    for max_q in HINTS:
        c.mass.fill_(7)
        tab = table(pkg, [dict(seqs[0], mass=c.mass[0].data_ptr() + off), seqs[1]], c, [0, 1], mass=True)
        assert gpu_lib.d1_kv4_mass(P(dx), dx.shape[1], P(l), len(x), P(tab), 2, max_q, 140, 4, 2, 0.125, 0, len(x), ST()) == 0
        assert gpu_lib.d1_kv4_error() != 0
        got = c.mass.double().cpu().numpy()
        assert (got[0] == 7).all() and (np.abs(got - M) <= T)[1, :, :40].all()
    mass, kept = torch.rand(2, 2, 144, device="cuda"), torch.zeros(2, 2, 24, dtype=torch.int32, device="cuda")
    for bad in (dict(mass=P(mass) + off), dict(dst_mass=P(d.mass) + off), dict(kept=P(kept) + off)):
        arr = (pkg.abi.Kv4Evict * 2)()
        for i, e in enumerate(arr):
            e.len, e.cap, e.keep, e.recent, e.dst_cap, e.mass = 40, c.cap, 20, 2, d.cap, mass[i].data_ptr()
            e.dst_mass, e.kept = d.mass[i].data_ptr(), kept[i].data_ptr()
            for k in c.dev:
                setattr(e, k, c.dev[k][i].data_ptr())
                setattr(e, "dst_" + k, d.dev[k][i].data_ptr())
        for k, v in bad.items():
            setattr(arr[0], k, v)
        items = torch.frombuffer(bytearray(bytes(arr)), dtype=torch.uint8).cuda()
        d.dev["kp"].fill_(77)
        assert gpu_lib.d1_kv4_evict(P(items), 2, 40, 2, ST()) == 0 and gpu_lib.d1_kv4_error() != 0
        assert (d.dev["kp"][0] == 77).all() and (d.dev["kp"][1, :, :20] != 77).all()


@gpu
def test_evict_bad_items_are_skipped(pkg, gpu_lib):
    rng = np.random.default_rng(7)
    c, d = Caches(rng, [40, 40], 2), Caches(rng, [0, 0], 2, 24)
    mass = torch.rand(2, 2, 40, device="cuda")
    for bad in (dict(keep=30), dict(keep=-1), dict(recent=-1), dict(len=41), dict(len=-1), dict(cap=36), dict(dst_cap=20),
                dict(mass=None), dict(k4=None), dict(dst_vp=None), dict(dst_k4=d.dev["k4"].data_ptr() + 4)):
        arr = (pkg.abi.Kv4Evict * 2)()
        for i in range(2):
            e = arr[i]
            e.len, e.cap, e.keep, e.recent, e.dst_cap, e.mass = 40, c.cap, 20, 2, d.cap, mass[i].data_ptr()
            for k in c.dev:
                setattr(e, k, c.dev[k][i].data_ptr())
                setattr(e, "dst_" + k, d.dev[k][i].data_ptr())
        for k, v in bad.items():
            setattr(arr[0], k, v)
        items = torch.frombuffer(bytearray(bytes(arr)), dtype=torch.uint8).cuda()
        d.dev["kp"].fill_(77)
        assert gpu_lib.d1_kv4_evict(P(items), 2, 40, 2, ST()) == 0
        assert gpu_lib.d1_kv4_error() != 0
        assert (d.dev["kp"][0] == 77).all() and (d.dev["kp"][1, :, :20] != 77).all()


@gpu
@pytest.mark.parametrize("max_q", HINTS)
def test_far_heads(pkg, gpu_lib, max_q):
    """A kv head whose codes lie behind the 32-bit range of its arrays (the arrays are not initialised elsewhere)."""
    kvh, group, cap, n, off = 5, 1, 2 ** 24 + 8, 70, 2 ** 24 - 70
    rng = np.random.default_rng(8)
    k4, v4 = (torch.empty(kvh, cap, 32, dtype=torch.uint8, device="cuda") for _ in range(2))
    kp, vp = (torch.zeros(kvh, cap, dtype=torch.int16, device="cuda") for _ in range(2))
    x = rng.standard_normal((n, 3 * kvh * 64)).astype(np.float16)
    d = torch.from_numpy(x).cuda()
    ptr = dict(k4=P(k4), v4=P(v4), kp=P(kp), vp=P(vp), ext_cap=cap)
    tab = table(pkg, [dict(kv_start=0, kv_len=n, ext_len=off, **ptr)])
    ld = 3 * kvh * 64
    assert gpu_lib.d1_kv4_append(d[:, kvh * 64:].data_ptr(), d[:, 2 * kvh * 64:].data_ptr(), ld, P(tab), 1, n, kvh, ST()) == 0
    y = torch.zeros(n, 2 * kvh * 64, dtype=torch.float16, device="cuda")
    assert gpu_lib.d1_kv4_load(P(tab), 1, n, kvh, P(y), y[:, kvh * 64:].data_ptr(), 2 * kvh * 64, ST()) == 0
    want = values(*pack(x.reshape(n, 3, kvh, 64)[:, 1:])).reshape(n, -1)
    assert (y.double().cpu().numpy() == want).all()
    # the same rows at the front of each head, and attended to
    tab = table(pkg, [dict(kv_start=0, kv_len=n, ext_len=0, **ptr)])
    assert gpu_lib.d1_kv4_append(d[:, kvh * 64:].data_ptr(), d[:, 2 * kvh * 64:].data_ptr(), ld, P(tab), 1, n, kvh, ST()) == 0
    c = Caches(rng, [n], kvh)
    for j, (a, p) in enumerate((("k4", "kp"), ("v4", "vp"))):
        c.host[a][0, :, :n], c.host[p][0, :, :n] = pack(x.reshape(n, 3, kvh, 64)[:, 1 + j].transpose(1, 0, 2))
    seqs = [dict(q_start=0, q_len=n, kv_start=0, kv_len=0)]
    O, L = attend(gpu_lib, d, table(pkg, [dict(seqs[0], ext_len=n, **ptr)]), 1, kvh, group, 0.125, max_q, n)
    assert gpu_lib.d1_kv4_error() == 0
    check_attend(O, L, plain_attend(x, seqs, c, [0], kvh, group, 0.125, True), kvh)


# ------------------------------------------------------------------------------------------------ together
class Step:
    """One layer as a server runs it: rows into the cache, attention over it, the weights, eviction, attention over what
    was kept."""

    def __init__(self, pkg, lib, seed, kvh=4, group=2, lens=(150, 37), rows=(40, 40), keep=64):
        rng = np.random.default_rng(seed)
        self.lib, self.kvh, self.group, self.keep, self.rows = lib, kvh, group, keep, rows
        self.c, self.d = Caches(rng, list(lens), kvh, 200), Caches(rng, [0, 0], kvh, keep)
        self.x, st = poisoned_rows(rng, rows, (kvh * group + 2 * kvh) * 64)
        self.dx, h, T = torch.from_numpy(self.x).cuda(), kvh * group, len(self.x)
        self.seqs = [dict(q_start=s, q_len=n, kv_start=s, kv_len=n) for s, n in zip(st, rows)]
        self.t0 = table(pkg, self.seqs, self.c, [0, 1])
        total = [a + b for a, b in zip(lens, rows)]
        own = [dict(s, kv_len=0) for s in self.seqs]
        self.t1 = table(pkg, [dict(s, ext_len=n) for s, n in zip(own, total)], self.c, [0, 1], mass=True)
        self.t2 = table(pkg, [dict(s, ext_len=min(keep, n)) for s, n in zip(own, total)], self.d, [0, 1])
        arr = (pkg.abi.Kv4Evict * 2)()
        for i in range(2):
            e = arr[i]
            e.len, e.cap, e.keep, e.recent, e.dst_cap, e.mass = total[i], self.c.cap, keep, 8, self.d.cap, self.c.mass[i].data_ptr()
            for k in self.c.dev:
                setattr(e, k, self.c.dev[k][i].data_ptr())
                setattr(e, "dst_" + k, self.d.dev[k][i].data_ptr())
        self.items = torch.frombuffer(bytearray(bytes(arr)), dtype=torch.uint8).cuda()
        self.total = total
        self.o1, self.o2 = (torch.zeros(T, h * 64, dtype=torch.float16, device="cuda") for _ in range(2))
        self.l1, self.l2 = (torch.zeros(h, T, device="cuda") for _ in range(2))

    def run(self, max_q):
        h, T, d, st = self.kvh * self.group, len(self.x), self.dx, ST()
        k, v, ld = d[:, h * 64:].data_ptr(), d[:, (h + self.kvh) * 64:].data_ptr(), d.shape[1]
        L = self.lib
        assert L.d1_kv4_append(k, v, ld, P(self.t0), 2, max(self.rows), self.kvh, st) == 0
        for tab, o, l in ((self.t1, self.o1, self.l1), (self.t2, self.o2, self.l2)):
            assert L.d1_flash_attn_kv4(P(d), ld, k, v, ld, P(o), h * 64, P(l), T, P(tab), 2, max_q, 190, h, self.group, 0.125,
                                       T, T, st) == 0
            if o is self.o1:
                assert L.d1_kv4_mass(P(d), ld, P(l), T, P(tab), 2, max_q, 190, h, self.group, 0.125, 0, T, st) == 0
                assert L.d1_kv4_evict(P(self.items), 2, 190, self.kvh, st) == 0

    def check(self):
        h = self.kvh * self.group
        q = [slice(s["q_start"], s["q_start"] + s["q_len"]) for s in self.seqs]
        for c, tot, o, l in ((self.c, self.total, self.o1, self.l1), (self.d, [min(self.keep, n) for n in self.total], self.o2, self.l2)):
            c.host, c.lens = c.back(), tot
            want = plain_attend(self.x, [dict(s, kv_len=0) for s in self.seqs], c, [0, 1], self.kvh, self.group, 0.125, True)
            for r in q:
                assert (np.abs(o.double().cpu().numpy()[r] - want[0][r]) <= want[2][r]).all()
                assert (np.abs(l.double().cpu().numpy()[:, r] - want[1][:, r]) <= want[3][:, r]).all()
        # the weights of a row's keys sum to 1, and what was kept is what the weights say
        m = self.c.mass.cpu().numpy()
        for i, n in enumerate(self.total):
            assert np.abs(m[i, :, :n].sum(-1) / (self.rows[i] * self.group) - 1).max() < 1e-4
            for g in range(self.kvh):
                at = keep_set(m[i, g, :n], self.keep, 8)
                assert (self.d.host["k4"][i, g, :len(at)] == self.c.host["k4"][i, g, at]).all()


@gpu
@pytest.mark.parametrize("max_q", HINTS)
def test_step_together(pkg, gpu_lib, max_q):
    s = Step(pkg, gpu_lib, 11)
    s.run(max_q)
    torch.cuda.synchronize()
    assert gpu_lib.d1_kv4_error() == 0
    s.check()


@gpu
@pytest.mark.parametrize("max_q", HINTS)
def test_step_captured_and_on_two_streams(pkg, gpu_lib, max_q):
    """The same step captured into two graphs, replayed at once on two streams, and again with other rows in place: the
    results of the eager step, bit for bit."""
    steps = [Step(pkg, gpu_lib, 21), Step(pkg, gpu_lib, 22)]
    other = Step(pkg, gpu_lib, 23)
    want = []
    for s in steps + [other]:
        s.run(max_q)
        torch.cuda.synchronize()
        want.append([s.o1.clone(), s.l1.clone(), s.o2.clone(), s.l2.clone(), s.c.mass.clone()])
    streams, graphs = [torch.cuda.Stream() for _ in range(2)], []
    for s, st in zip(steps, streams):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            s.run(max_q)
        graphs.append(g)
    for _ in range(3):
        for s in steps:
            for t in (s.o1, s.l1, s.o2, s.l2):
                t.fill_(0)
        torch.cuda.synchronize()
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        for s, w in zip(steps, want):
            for a, b in zip((s.o1, s.l1, s.o2, s.l2, s.c.mass), w):
                assert torch.equal(a.nan_to_num(9), b.nan_to_num(9))
    steps[0].dx.copy_(other.dx)
    for k in steps[0].c.dev:
        steps[0].c.dev[k].copy_(other.c.dev[k])
    with torch.cuda.stream(streams[0]):
        streams[0].wait_stream(torch.cuda.default_stream())
        graphs[0].replay()
    torch.cuda.synchronize()
    for a, b in zip((steps[0].o1, steps[0].l1, steps[0].o2, steps[0].l2, steps[0].c.mass), want[2]):
        assert torch.equal(a.nan_to_num(9), b.nan_to_num(9))
    assert gpu_lib.d1_kv4_error() == 0


@gpu
@pytest.mark.parametrize("max_q", HINTS)
def test_step_with_all_rows_cached(pkg, gpu_lib, max_q):
    """A server's step: rows appended, counted in ext_len, and kv_len = 0 with kv_start left where they were; the attention
    is called without K and V. Nor does it matter where a sequence without query rows starts."""
    rng = np.random.default_rng(31)
    kvh, group, rows, ext = 2, 2, [5, 0, 130, 33, 1], [3, 9, 200, 64, 0]
    h, n, total = kvh * group, 5, [a + b for a, b in zip(rows, ext)]
    c = Caches(rng, ext, kvh, 336)
    x, starts = poisoned_rows(rng, rows, (h + 2 * kvh) * 64)
    T, ld, d, lib = len(x), x.shape[1], torch.from_numpy(x).cuda(), gpu_lib
    seqs = [dict(q_start=s, q_len=m, kv_start=s, kv_len=m) for s, m in zip(starts, rows)]
    k, v = d[:, h * 64:].data_ptr(), d[:, (h + kvh) * 64:].data_ptr()
    assert lib.d1_kv4_append(k, v, ld, P(table(pkg, seqs, c, range(n))), n, max(rows), kvh, ST()) == 0
    c.lens, c.host = total, c.back()
    seqs = [dict(s, kv_len=0) for s in seqs]
    seqs[1].update(q_start=10 ** 6, kv_start=-7)
    tab = table(pkg, seqs, c, range(n), mass=True)
    O, L = torch.full((T, h * 64), 7.0, dtype=torch.float16, device="cuda"), torch.full((h, T), 7.0, device="cuda")
    assert lib.d1_flash_attn_kv4(P(d), ld, None, None, 0, P(O), h * 64, P(L), T, P(tab), n, max_q, max(total), h, group, 0.125,
                                 T, 0, ST()) == 0
    assert lib.d1_kv4_mass(P(d), ld, P(L), T, P(tab), n, max_q, max(total), h, group, 0.125, 0, T, ST()) == 0
    assert lib.d1_kv4_append(k, v, ld, P(tab), n, max(rows), kvh, ST()) == 0 and lib.d1_kv4_error() == 0
    seqs[1].update(q_start=0, kv_start=0)
    check_attend(O, L, plain_attend(x, seqs, c, range(n), kvh, group, 0.125, True), h)
    lse = L.cpu().numpy()
    M, tol = plain_mass(x, lse, seqs, c, range(n), kvh, group, 0.125)
    got = c.mass.double().cpu().numpy()
    assert all((np.abs(got - M) <= tol)[i, :, :m].all() for i, m in enumerate(total))


@gpu
@pytest.mark.parametrize("heads,group", [(2 ** 25, 2 ** 13), (2 ** 26, 2 ** 14), (2 ** 30, 2 ** 20)])
def test_heads_beyond_32_bits_are_refused(pkg, gpu_lib, heads, group):
    """64 columns a head would not be countable in 32 bits: refused, whatever the leading dimension."""
    tab, d = table(pkg, [dict(q_len=0)]), torch.zeros(8, 64, dtype=torch.float16, device="cuda")
    lse = torch.zeros(8, device="cuda")
    for max_q in (1, 5000):
        assert gpu_lib.d1_flash_attn_kv4(P(d), 64, None, None, 0, P(d), 64, None, 0, P(tab), 1, max_q, 1, heads, group, 0.125, 1, 0,
                                         ST()) == -1
        assert gpu_lib.d1_kv4_mass(P(d), 64, P(lse), 8, P(tab), 1, max_q, 1, heads, group, 0.125, 0, 1, ST()) == -1
    torch.cuda.synchronize()
    assert gpu_lib.d1_kv4_error() == 0


@gpu
@pytest.mark.parametrize("max_q", HINTS)
def test_server_loop(pkg, gpu_lib, max_q):
    """A bounded cache over three steps: append, the new keys' weights set to 0 by the caller, attention, weights added up
    over the steps, eviction into the other cache."""
    rng = np.random.default_rng(32)
    kvh, group, keep, lib = 2, 2, 64, gpu_lib
    h, n, lens, rows = kvh * group, 2, [150, 0], [40, 70]
    a, b = Caches(rng, lens, kvh, 240), Caches(rng, [0, 0], kvh, 240)
    a.mass[:] = float("nan")
    for i, m in enumerate(lens):
        a.mass[i, :, :m] = 0
    sums, tols = np.zeros((n, kvh, 240)), np.zeros((n, kvh, 240))
    for step in range(3):
        x, starts = poisoned_rows(rng, rows, (h + 2 * kvh) * 64)
        d, T = torch.from_numpy(x).cuda(), len(x)
        k, v, ld = d[:, h * 64:].data_ptr(), d[:, (h + kvh) * 64:].data_ptr(), x.shape[1]
        seqs = [dict(q_start=s, q_len=m, kv_start=s, kv_len=m) for s, m in zip(starts, rows)]
        assert lib.d1_kv4_append(k, v, ld, P(table(pkg, seqs, a, range(n))), n, max(rows), kvh, ST()) == 0
        for i in range(n):
            a.mass[i, :, a.lens[i]:a.lens[i] + rows[i]] = 0
        a.lens, a.host = [p + q for p, q in zip(a.lens, rows)], a.back()
        tab = table(pkg, [dict(s, kv_len=0) for s in seqs], a, range(n), mass=True)
        O, L = torch.zeros(T, h * 64, dtype=torch.float16, device="cuda"), torch.zeros(h, T, device="cuda")
        assert lib.d1_flash_attn_kv4(P(d), ld, None, None, 0, P(O), h * 64, P(L), T, P(tab), n, max_q, max(a.lens), h, group, 0.125,
                                     T, 0, ST()) == 0
        assert lib.d1_kv4_mass(P(d), ld, P(L), T, P(tab), n, max_q, max(a.lens), h, group, 0.125, 1, T, ST()) == 0
        arr = (pkg.abi.Kv4Evict * n)()
        for i, e in enumerate(arr):
            e.len, e.cap, e.keep, e.recent, e.dst_cap = a.lens[i], a.cap, keep, 8, b.cap
            e.mass, e.dst_mass = a.mass[i].data_ptr(), b.mass[i].data_ptr()
            for f in a.dev:
                setattr(e, f, a.dev[f][i].data_ptr())
                setattr(e, "dst_" + f, b.dev[f][i].data_ptr())
        items = torch.frombuffer(bytearray(bytes(arr)), dtype=torch.uint8).cuda()
        assert lib.d1_kv4_evict(P(items), n, max(a.lens), kvh, ST()) == 0 and lib.d1_kv4_error() == 0
        own = [dict(s, kv_len=0) for s in seqs]
        want = plain_attend(x, own, a, range(n), kvh, group, 0.125, True)
        M, tol = plain_mass(x, L.cpu().numpy(), own, a, range(n), kvh, group, 0.125)
        got, moved, back = a.mass.cpu().numpy(), b.mass.cpu().numpy(), b.back()
        nsum, ntol = np.zeros_like(sums), np.zeros_like(tols)
        for i, m in enumerate(a.lens):
            r = slice(starts[i], starts[i] + rows[i])
            assert (np.abs(O.double().cpu().numpy()[r] - want[0][r]) <= want[2][r]).all()
            all_, t = sums[i, :, :m] + M[i, :, :m], tols[i, :, :m] + tol[i, :, :m]
            t += 2.0 ** -24 * all_  # the addition
            assert (np.abs(got[i, :, :m] - all_) <= t).all()
            for g in range(kvh):
                at = keep_set(got[i, g, :m], keep, 8)
                assert (moved[i, g, :len(at)] == got[i, g, at]).all() and (back["k4"][i, g, :len(at)] == a.host["k4"][i, g, at]).all()
                nsum[i, g, :len(at)], ntol[i, g, :len(at)] = all_[g, at], t[g, at]
        sums, tols = nsum, ntol
        b.lens = [min(keep, m) for m in a.lens]
        a, b = b, a


# ------------------------------------------------------------------------------------------------ units after units
# (queries, cached keys, own rows, kv heads, group): more units than CTAs, so that a CTA goes from one to the next
UNITS = {
    # heads without a partner, blocks of 256 rows and what is left of them: a block with rows for one warpgroup alone, then
    # one with rows for both, whose keys are cached, own, or both
    "one warpgroup, then both": ([300] * 10, [1000, 0, 1000, 130, 999, 0, 520, 1000, 3, 1000],
                                 [300, 700, 0, 300, 300, 1, 0, 700, 300, 0], 16, 1),
    "one warpgroup, then packed": ([300, 129, 100, 7, 290, 260, 90, 300, 128, 40] * 3, [1000, 300, 700, 0, 600, 129] * 5,
                                   [0, 0, 300, 7, 129, 1, 700, 640, 0, 40] * 3, 16, 1),
    "three heads": ([280 + 7 * (i % 5) if i % 3 else 40 for i in range(40)], [1000 * (i % 2) + i for i in range(40)],
                    [(0, 300, 700)[i % 3] for i in range(40)], 3, 3),
    # partial tiles of own rows one after the other, with nothing cached before them
    "own rows only": ([60 - i % 20 for i in range(300)], [0] * 300, [60 - i % 20 for i in range(300)], 4, 2),
    "few own rows": ([40 + i % 9 for i in range(300)], [128 * (i % 5 == 0) for i in range(300)], [1 + i % 130 for i in range(300)], 4, 2),
    # full packed units, which both warpgroups read, before and after blocks that leave some warps without rows
    "warps without rows": ([(64, 130, 64, 1, 165, 200)[i % 6] for i in range(60)], [(900, 300, 129, 640, 260, 0)[i % 6] for i in range(60)],
                           [(0, 1, 300, 0, 0, 129)[i % 6] for i in range(60)], 4, 2),
}


@gpu
@pytest.mark.parametrize("exact_hint", [True, False])
@pytest.mark.parametrize("name", UNITS)
def test_attend_units_in_turn(pkg, gpu_lib, name, exact_hint):
    """CTAs that take unit after unit of every kind, at their full number and, by a hint just above 64 packed rows, fewer:
    right, and the same bits each time."""
    q, ext, kv, kvh, group = UNITS[name]
    n, h = len(q), kvh * group
    rng = np.random.default_rng(len(name) + 70)
    c = Caches(rng, ext, kvh, -(-max(ext) // 8) * 8)
    x, starts = poisoned_rows(rng, [max(a, b) for a, b in zip(q, kv)], (h + 2 * kvh) * 64)
    seqs = [dict(q_start=s, q_len=a, kv_start=s, kv_len=b) for s, a, b in zip(starts, q, kv)]
    want = plain_attend(x, seqs, c, list(range(n)), kvh, group, 0.125, True)
    tab, d, first = table(pkg, seqs, c, range(n)), torch.from_numpy(x).cuda(), None
    for _ in range(4):
        O, L = attend(gpu_lib, d, tab, n, kvh, group, 0.125, max(q) if exact_hint else 64 // group + 1,
                      max(a + b for a, b in zip(ext, kv)))
        assert gpu_lib.d1_kv4_error() == 0
        if first is None:
            check_attend(O, L, want, h)
            first = O, L
        assert torch.equal(O, first[0]) and torch.equal(L, first[1])
