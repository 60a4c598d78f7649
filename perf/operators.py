"""Workloads of the 4-bit key/value cache operators (include/d1kernels.h, d1_kv4_*), with their plain forms.

A cache holds the keys and values that a sequence attends to before its own rows (a media prefix, or the rows of
earlier steps), 64 dimensions per kv head, each vector as 64 codes of 4 bits and one 16-bit parameter:
    lo = min(0, min x), hi = max(0, max x)
    step = (hi - lo) / 15 rounded up to 7 significant bits (a multiple of 2^-20), zero = round(-lo / step) in 0..15
    code = round(x / step) + zero in 0..15, with |code - zero| * step within fp16; the vector stands for
    (code - zero) * step, which fp16 holds exactly.
The parameter is step's fp16 bits, whose low 4 bits are free and hold zero. Code 8w + 2n of a vector is at bits 4n of
its 32-bit word w, code 8w + 2n + 1 at bits 16 + 4n.

Operators:
    append   rows of fp16 keys and values into the caches of a batch, and those rows read back (d1_kv4_append, d1_kv4_load)
    attend   softmax attention of packed rows over [cached keys | the sequence's own fp16 rows], with each row's
             log-sum-exp (d1_flash_attn_kv4)
    mass     the attention weight that each cached key received, summed over the rows and the heads of its kv head
             (d1_kv4_mass)
    evict    of each kv head, the keys with the most weight and the most recent ones, in their order, into another
             cache, with their weights; and the kept rows read back (d1_kv4_evict, d1_kv4_load)
"""
import math
import random
import sys

import numpy as np
import torch

own = False

HD = 64  # dimensions per head
# D1Kv4Seq and D1Kv4Evict of include/d1kernels.h
SEQ = np.dtype([("q_start", "<i4"), ("q_len", "<i4"), ("kv_start", "<i4"), ("kv_len", "<i4"), ("ext_len", "<i4"),
                ("ext_cap", "<i4"), ("k4", "<u8"), ("v4", "<u8"), ("kp", "<u8"), ("vp", "<u8"), ("mass", "<u8")])
EVICT = np.dtype([("len", "<i4"), ("cap", "<i4"), ("keep", "<i4"), ("recent", "<i4"), ("dst_cap", "<i4"), ("pad", "<i4"),
                  ("k4", "<u8"), ("v4", "<u8"), ("kp", "<u8"), ("vp", "<u8"), ("mass", "<u8"),
                  ("dst_k4", "<u8"), ("dst_v4", "<u8"), ("dst_kp", "<u8"), ("dst_vp", "<u8"), ("dst_mass", "<u8"),
                  ("kept", "<u8")])


def listed():
    # the trunk's attention: 16 query heads, 8 kv heads; the decision head's: 16 and 16
    t = {"kvh": 8, "group": 2}
    return [
        # one new row in each of 16 conversations: the latency of a step
        {"name": "append step", "op": "append", "caches": 16, "rows": 1, "ext": 1024, "ragged": True, **t},
        # one image's prefix, an odd number of rows
        {"name": "append prefix", "op": "append", "caches": 1, "rows": 1025, "ext": 0, "ragged": False, **t},
        # a full batch of long media prefixes
        {"name": "append batch", "op": "append", "caches": 8, "rows": 4096, "ext": 0, "ragged": True, **t},
        # a single token over one long cache: everything is latency and the split over the keys
        {"name": "attend token", "op": "attend", "seqs": 1, "share": 1, "q": 1, "ext": 4097, "local": True,
         "ragged": False, **t},
        # decoding for 32 requests at the longest context: bound by the cache's bytes
        {"name": "attend decode", "op": "attend", "seqs": 32, "share": 1, "q": 1, "ext": 16384, "local": True,
         "ragged": True, **t},
        # short questions about a shared medium, with their own rows behind it, as the engine packs them
        {"name": "attend questions", "op": "attend", "seqs": 48, "share": 6, "q": 45, "ext": 1200, "local": True,
         "ragged": True, **t},
        # long documents after a long prefix: bound by the matrix and exponential units
        {"name": "attend documents", "op": "attend", "seqs": 4, "share": 1, "q": 2048, "ext": 4096, "local": True,
         "ragged": True, **t},
        # the weights that short questions give the keys of a long cache
        {"name": "mass questions", "op": "mass", "seqs": 8, "share": 2, "q": 24, "ext": 4100, "ragged": True, **t},
        # the weights that a document's rows give the keys before it
        {"name": "mass documents", "op": "mass", "seqs": 2, "share": 1, "q": 2048, "ext": 8192, "ragged": True, **t},
        # one layer of a medium-sized prefix, half of it kept
        {"name": "evict prefix", "op": "evict", "caches": 1, "ext": 1500, "keep": 750, "recent": 33, "ragged": False,
         **t},
        # the six attention layers of four long caches, a quarter of them kept
        {"name": "evict long", "op": "evict", "caches": 24, "ext": 16384, "keep": 4096, "recent": 64, "ragged": True,
         **t},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "mass", "evict"])
    kvh, group = rng.choice([(8, 2), (8, 2), (16, 1), (4, 4), (3, 3), (2, 8)])
    c = {"op": op, "kvh": kvh, "group": group, "ragged": rng.random() < 0.7}
    if op == "append":
        rows = _log_int(rng, 1, 4096)
        c.update(rows=rows, caches=_log_int(rng, 1, max(1, min(32, 32768 // rows))), ext=_log_int(rng, 1, 4096) - 1)
    elif op in ("attend", "mass"):
        q, ext = _log_int(rng, 1, 2048), _log_int(rng, 1, 16384)
        most = max(1, min(32, int(2 ** 25 / (q * (ext + q))), int(2 ** 19 / ext)))
        seqs = _log_int(rng, 1, most)
        c.update(seqs=seqs, share=rng.choice([1, 1, 2, 5]), q=q, ext=ext)
        if op == "attend":
            c["local"] = rng.random() < 0.8
    else:
        ext = _log_int(rng, 2, 16384)
        c.update(caches=_log_int(rng, 1, 24), ext=ext, keep=_log_int(rng, 1, ext), recent=_log_int(rng, 1, 65) - 1)
    return c


def _lens(case):
    """Lengths of the case's sequences and caches: they follow from the case, not from the seed."""
    r = random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))
    vary = lambda n, lo=1: r.randint(max(lo, n // 2), n) if case["ragged"] else n  # noqa: E731
    op = case["op"]
    if op == "append":
        return {"rows": [vary(case["rows"]) for _ in range(case["caches"])],
                "ext": [vary(case["ext"], 0) if case["ext"] else 0 for _ in range(case["caches"])]}
    if op == "evict":
        return {"ext": [vary(case["ext"]) for _ in range(case["caches"])]}
    caches = -(-case["seqs"] // case["share"])
    return {"q": [vary(case["q"]) for _ in range(case["seqs"])], "ext": [vary(case["ext"]) for _ in range(caches)],
            "of": [i // case["share"] for i in range(case["seqs"])]}


def _starts(lens):
    return [0] + list(np.cumsum(lens))[:-1]


def _up8(n):
    return -(-n // 8) * 8


# ------------------------------------------------------------------------------------------------ the cache format
def _quantise(x):
    """fp16 [..., 64] -> codes (int32), step and zero (fp32, [..., 1])."""
    x = x.float()
    lo, hi = x.amin(-1, keepdim=True).clamp(max=0), x.amax(-1, keepdim=True).clamp(min=0)
    step = (hi - lo) / torch.full_like(lo, 15.0)
    exp2 = torch.frexp(step)[1]
    unit = ((exp2 - 7).clamp(min=-20) + 127).bitwise_left_shift(23).view(torch.float32)  # a power of two
    step = torch.ceil(step / unit) * unit
    s = torch.where(step > 0, step, torch.ones_like(step))
    zero = torch.round(-lo / s).clamp(0, 15)
    top = torch.floor(torch.full_like(s, 65504.0) / s)
    code = torch.maximum(torch.minimum(torch.round(x / s), top), -top) + zero
    return code.clamp(0, 15).int(), step, zero


def _values(code, step, zero):
    return (code.float() - zero) * step


def _pack(code, step, zero):
    """codes [..., 64], step, zero [..., 1] -> bytes [..., 32], parameters [...] (int16 bits)."""
    c = code.view(*code.shape[:-1], 8, 4, 2)
    at = torch.arange(4, device=c.device, dtype=torch.int32) * 4
    half = c.bitwise_left_shift(at[:, None]).sum(-2, dtype=torch.int32)  # [..., 8, 2]: the two halves of each word
    half = torch.where(half > 32767, half - 65536, half).to(torch.int16)
    par = step.half().view(torch.int16).bitwise_or(zero.to(torch.int16)).squeeze(-1)
    return half.contiguous().view(torch.uint8).reshape(*code.shape[:-1], 32), par


def _unpack(b, par):
    """bytes [..., 32], parameters [...] -> the fp32 values they stand for."""
    half = b.contiguous().view(torch.int16).int().bitwise_and(0xFFFF)  # [..., 16]: words' low and high halves
    at = torch.arange(4, device=b.device, dtype=torch.int32) * 4
    c = half.view(*half.shape[:-1], 8, 1, 2).bitwise_right_shift(at[:, None]).bitwise_and(15)
    c = c.reshape(*half.shape[:-1], 64)
    zero = par.bitwise_and(15).float().unsqueeze(-1)
    step = par.bitwise_and(-16).view(torch.float16).float().unsqueeze(-1)
    return _values(c, step, zero)


# ------------------------------------------------------------------------------------------------ inputs
def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _keys(g, kvh, rows):
    """Keys and values as the trunk's: keys with channels of unequal size, values with a few large entries."""
    chan = torch.exp(0.5 * _randn(g, kvh, 1, HD))
    k = _randn(g, kvh, rows, HD) * chan
    v = _randn(g, kvh, rows, HD) * torch.exp(0.3 * _randn(g, kvh, rows, 1))
    return k.half(), v.half()


def _caches(g, lens, cap, kvh):
    """Packed caches of the given lengths: [cache, kv head, cap] rows, zero behind a cache's last one."""
    n = len(lens)
    s = {"k4": torch.zeros(n, kvh, cap, 32, dtype=torch.uint8, device="cuda"),
         "kp": torch.zeros(n, kvh, cap, dtype=torch.int16, device="cuda")}
    s["v4"], s["vp"] = torch.zeros_like(s["k4"]), torch.zeros_like(s["kp"])
    for i, m in enumerate(lens):
        if m:
            k, v = _keys(g, kvh, m)
            s["k4"][i, :, :m], s["kp"][i, :, :m] = _pack(*_quantise(k))
            s["v4"][i, :, :m], s["vp"][i, :, :m] = _pack(*_quantise(v))
    return s


def _seq_table(n, q, qs, kv, ks, ext, cap, of, c, mass=None):
    t = np.zeros(n, SEQ)
    t["q_start"], t["q_len"], t["kv_start"], t["kv_len"], t["ext_len"], t["ext_cap"] = qs, q, ks, kv, ext, cap
    for name in ("k4", "v4", "kp", "vp"):
        t[name] = c[name].data_ptr() + np.asarray(of, np.uint64) * np.uint64(c[name][0].numel() * c[name].element_size())
    if mass is not None:
        t["mass"] = mass.data_ptr() + np.asarray(of, np.uint64) * np.uint64(mass[0].numel() * 4)
    return torch.frombuffer(bytearray(t.tobytes()), dtype=torch.uint8).cuda()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    kvh, group, L = case["kvh"], case["group"], _lens(case)
    s = {"op": case["op"], "kvh": kvh, "group": group, "heads": kvh * group, "scale": HD ** -0.5}
    dev = lambda v: torch.tensor(v, device="cuda", dtype=torch.int64)  # noqa: E731
    if s["op"] == "append":
        n, T, cap = len(L["rows"]), sum(L["rows"]), _up8(max(a + b for a, b in zip(L["rows"], L["ext"])))
        k, v = _keys(g, kvh, T)
        # rows of a fused projection [q | k | v], as the trunk's
        qkv = torch.empty(T, (s["heads"] + 2 * kvh) * HD, dtype=torch.float16, device="cuda")
        qkv.normal_(generator=g)
        qkv[:, s["heads"] * HD:] = torch.cat([k, v]).transpose(0, 1).reshape(T, -1)
        c = _caches(g, L["ext"], cap, kvh)
        st = _starts(L["rows"])
        s.update(c, qkv=qkv, n=n, ld=qkv.shape[1], max_rows=max(L["rows"]),
                 cache=torch.repeat_interleave(dev(range(n)), dev(L["rows"])),
                 at=torch.arange(T, device="cuda") - torch.repeat_interleave(dev(st) - dev(L["ext"]), dev(L["rows"])),
                 seqs=_seq_table(n, 0, 0, L["rows"], st, L["ext"], cap, range(n), c),
                 ok=torch.empty(T, kvh * HD, dtype=torch.float16, device="cuda"),
                 ov=torch.empty(T, kvh * HD, dtype=torch.float16, device="cuda"))
    elif s["op"] in ("attend", "mass"):
        n, T, cap = len(L["q"]), sum(L["q"]), _up8(max(L["ext"]))
        c, st = _caches(g, L["ext"], cap, kvh), _starts(L["q"])
        qkv = torch.empty(T, (s["heads"] + 2 * kvh) * HD, dtype=torch.float16, device="cuda")
        qkv.normal_(generator=g)
        ext = [L["ext"][i] for i in L["of"]]
        local = bool(case.get("local"))
        kv = L["q"] if local else [0] * n
        mass = None
        if s["op"] == "mass":
            mass = torch.zeros(len(L["ext"]), kvh, cap, device="cuda")
            # log-sum-exps of the size that an attention over these keys gives
            s["lse"] = torch.log(torch.repeat_interleave(dev(ext), dev(L["q"])).float()) + 1 + 0.5 * _randn(g, s["heads"], T)
            s["mass"] = mass
        else:
            s["o"] = torch.empty(T, s["heads"] * HD, dtype=torch.float16, device="cuda")
            s["lse"] = torch.empty(s["heads"], T, device="cuda")
        s.update(c, qkv=qkv, n=n, T=T, ld=qkv.shape[1], max_q=max(L["q"]), max_ext=max(L["ext"]),
                 max_keys=max(a + b for a, b in zip(ext, kv)), q_start=dev(st), q_len=dev(L["q"]), kv_len=dev(kv),
                 ext_len=dev(L["ext"]), of=dev(L["of"]), local=local,
                 seqs=_seq_table(n, L["q"], st, kv, st, ext, cap, L["of"], c, mass))
    else:
        n, cap = len(L["ext"]), _up8(max(L["ext"]))
        c = _caches(g, L["ext"], cap, kvh)
        # weights with many equal ones: of short questions, most keys have about none
        mass = torch.floor(torch.rand(n, kvh, cap, generator=g, device="cuda") ** 6 * 4096) / 64
        keep = [min(case["keep"], m) for m in L["ext"]]
        dcap = _up8(case["keep"])
        d = {"d_" + k: torch.zeros(n, kvh, dcap, *v.shape[3:], dtype=v.dtype, device="cuda") for k, v in c.items()}
        d["d_mass"] = torch.zeros(n, kvh, dcap, device="cuda")
        d["kept"] = torch.full((n, kvh, dcap), -1, dtype=torch.int32, device="cuda")
        t = np.zeros(n, EVICT)
        t["len"], t["cap"], t["keep"], t["recent"], t["dst_cap"] = L["ext"], cap, case["keep"], case["recent"], dcap
        for name, x in {**c, "mass": mass, **{"dst_" + k[2:]: v for k, v in d.items() if k != "kept"},
                        "kept": d["kept"]}.items():
            t[name] = x.data_ptr() + np.arange(n, dtype=np.uint64) * np.uint64(x[0].numel() * x.element_size())
        st, dc = _starts(keep), {k[2:]: v for k, v in d.items() if k.startswith("d_")}
        s.update(c, **d, mass=mass, n=n, cap=cap, max_ext=max(L["ext"]), max_keep=max(keep), keep=case["keep"],
                 recent=case["recent"], ext_len=dev(L["ext"]),
                 items=torch.frombuffer(bytearray(t.tobytes()), dtype=torch.uint8).cuda(),
                 cache=torch.repeat_interleave(dev(range(n)), dev(keep)),
                 at=torch.arange(sum(keep), device="cuda") - torch.repeat_interleave(dev(st), dev(keep)),
                 seqs=_seq_table(n, 0, 0, keep, st, 0, dcap, range(n), dc),
                 ok=torch.empty(sum(keep), kvh * HD, dtype=torch.float16, device="cuda"),
                 ov=torch.empty(sum(keep), kvh * HD, dtype=torch.float16, device="cuda"))
    return s


# ------------------------------------------------------------------------------------------------ plain forms
def _plain_append(s):
    h, kvh = s["heads"], s["kvh"]
    kv = s["qkv"][:, h * HD:].reshape(-1, 2, kvh, HD)
    b, par = _pack(*_quantise(kv))
    at = (s["cache"][:, None], torch.arange(kvh, device="cuda")[None], s["at"][:, None])
    s["k4"][at], s["v4"][at], s["kp"][at], s["vp"][at] = b[:, 0], b[:, 1], par[:, 0], par[:, 1]
    back = lambda x, p: _unpack(s[x][at], s[p][at]).half().reshape(-1, kvh * HD)  # noqa: E731
    return {"k": back("k4", "kp"), "v": back("v4", "vp")}


def _padded(s):
    """Row numbers of the sequences' rows, [sequence, max_q], and which of them there are."""
    i = torch.arange(s["max_q"], device="cuda")
    there = i < s["q_len"][:, None]
    return torch.where(there, s["q_start"][:, None] + i, 0), there


def _scores(s, row, key):
    """[sequence, kv head, group, row, key] of fp32."""
    q = s["qkv"][:, :s["heads"] * HD][row].float().view(*row.shape, s["kvh"], s["group"], HD)
    q = q.permute(0, 2, 3, 1, 4).flatten(2, 3)
    return (q @ key.transpose(-1, -2)).view(*q.shape[:2], s["group"], row.shape[1], -1) * s["scale"]


def _plain_attend(s):
    h, kvh = s["heads"], s["kvh"]
    row, there = _padded(s)
    cap = s["k4"].shape[2]
    key, val = _unpack(s["k4"], s["kp"])[s["of"]], _unpack(s["v4"], s["vp"])[s["of"]]  # [sequence, kv head, cap, 64]
    ok = torch.arange(cap, device="cuda") < s["ext_len"][s["of"]][:, None]
    if s["local"]:
        kv = s["qkv"][:, h * HD:][row].float().view(*row.shape, 2, kvh, HD).permute(2, 0, 3, 1, 4)
        key, val, ok = torch.cat([key, kv[0]], 2), torch.cat([val, kv[1]], 2), torch.cat([ok, there], 1)
    x = _scores(s, row, key).masked_fill(~ok[:, None, None, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    x = torch.exp(x - top)
    total = x.sum(-1, keepdim=True)
    o = (x / total).flatten(2, 3) @ val  # [sequence, kv head, group * row, 64]
    o = o.view(*x.shape[:4], HD).permute(0, 3, 1, 2, 4)[there].reshape(-1, h * HD)
    lse = (top + torch.log(total)).squeeze(-1).permute(0, 3, 1, 2)[there].reshape(-1, h)
    return {"o": o.half(), "lse": lse.t().contiguous()}


def _plain_mass(s):
    row, there = _padded(s)
    key = _unpack(s["k4"], s["kp"])[s["of"]]
    lse = s["lse"][:, row].view(s["kvh"], s["group"], *row.shape).permute(2, 0, 1, 3)[..., None]
    w = torch.exp(_scores(s, row, key) - lse) * there[:, None, None, :, None]
    w = w.sum((2, 3)) * (torch.arange(key.shape[2], device="cuda") < s["ext_len"][s["of"]][:, None])[:, None]
    return {"mass": torch.zeros_like(s["mass"]).index_add_(0, s["of"], w)}


def _plain_evict(s):
    n, kvh, cap = s["mass"].shape
    i, length = torch.arange(cap, device="cuda"), s["ext_len"][:, None, None]
    keep = length.clamp(max=s["keep"])
    recent = keep.clamp(max=s["recent"])
    cand = i < length - recent
    m = torch.where(cand & ~torch.isnan(s["mass"]), s["mass"], -math.inf)
    order = torch.sort(m, dim=-1, descending=True, stable=True)[1]
    chosen = torch.zeros(n, kvh, cap, dtype=torch.bool, device="cuda")
    chosen.scatter_(2, order, (i < keep - recent).expand(n, kvh, cap))
    chosen |= (i >= length - recent) & (i < length)
    at = torch.sort((~chosen).to(torch.uint8), dim=-1, stable=True)[1][..., :s["d_mass"].shape[2]]  # chosen ones first
    if at.shape[2] < s["d_mass"].shape[2]:
        at = torch.nn.functional.pad(at, (0, s["d_mass"].shape[2] - at.shape[2]))
    in_ = torch.arange(at.shape[2], device="cuda") < keep
    kept, mass = torch.where(in_, at, -1).int(), torch.where(in_, torch.gather(s["mass"], 2, at), 0)
    rows = lambda x: torch.where(in_[..., None], torch.gather(x, 2, at[..., None].expand(-1, -1, -1, 32)), 0)  # noqa: E731
    pars = lambda x: torch.where(in_, torch.gather(x, 2, at), 0)  # noqa: E731
    pick = (s["cache"][:, None], torch.arange(kvh, device="cuda")[None], s["at"][:, None])
    back = lambda x, p: _unpack(rows(s[x])[pick], pars(s[p])[pick]).half().reshape(-1, kvh * HD)  # noqa: E731
    return {"kept": kept, "mass": mass, "k": back("k4", "kp"), "v": back("v4", "vp")}


# ------------------------------------------------------------------------------------------------ the framework's
def _library():
    name = "fast_d1_omni_b200"
    if name not in sys.modules:
        import importlib.util
        from pathlib import Path
        at = Path(__file__).resolve().parents[1] / "fast-d1-omni_b200"
        spec = importlib.util.spec_from_file_location(name, at / "__init__.py", submodule_search_locations=[str(at)])
        sys.modules[name] = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(sys.modules[name])
    return sys.modules[name].lib(), sys.modules[name].check


def _own(s):
    lib, check = _library()
    p = lambda k: s[k].data_ptr()  # noqa: E731
    st, h, kvh, op = torch.cuda.current_stream().cuda_stream, s["heads"], s["kvh"], s["op"]
    if op == "evict":
        check(lib.d1_kv4_evict(p("items"), s["n"], s["max_ext"], kvh, st), "kv4_evict")
        check(lib.d1_kv4_load(p("seqs"), s["n"], s["max_keep"], kvh, p("ok"), p("ov"), kvh * HD, st), "kv4_load")
        return {"kept": s["kept"], "mass": s["d_mass"], "k": s["ok"], "v": s["ov"]}
    q, ld = p("qkv"), s["ld"]
    k, v = q + h * HD * 2, q + (h + kvh) * HD * 2
    if op == "append":
        check(lib.d1_kv4_append(k, v, ld, p("seqs"), s["n"], s["max_rows"], kvh, st), "kv4_append")
        check(lib.d1_kv4_load(p("seqs"), s["n"], s["max_rows"], kvh, p("ok"), p("ov"), kvh * HD, st), "kv4_load")
        return {"k": s["ok"], "v": s["ov"]}
    T = s["T"]
    if op == "attend":
        check(lib.d1_flash_attn_kv4(q, ld, k, v, ld, p("o"), h * HD, p("lse"), T, p("seqs"), s["n"], s["max_q"],
                                    s["max_keys"], h, s["group"], s["scale"], T, T, st), "flash_attn_kv4")
        return {"o": s["o"], "lse": s["lse"]}
    check(lib.d1_kv4_mass(q, ld, p("lse"), T, p("seqs"), s["n"], s["max_q"], s["max_ext"], h, s["group"], s["scale"], 0,
                          T, st), "kv4_mass")
    return {"mass": s["mass"]}


def run(s):
    if own:
        return _own(s)
    if s["op"] == "append":
        return _plain_append(s)
    if s["op"] == "attend":
        return _plain_attend(s)
    if s["op"] == "mass":
        return _plain_mass(s)
    return _plain_evict(s)


# ------------------------------------------------------------------------------------------------ what it has to do
VEC = 34  # bytes of a cached vector


def work(case):
    kvh, group, L = case["kvh"], case["group"], _lens(case)
    h = kvh * group
    if case["op"] == "append":
        T = sum(L["rows"])  # the rows' keys and values once, their cached form once, the values read back once
        return {"bytes": T * kvh * 2 * (2 * HD + VEC + 2 * HD), "flops": T * kvh * 2 * HD * 4}
    if case["op"] == "evict":
        kept = sum(min(case["keep"], m) for m in L["ext"])  # all weights; the kept rows read, written and read back
        return {"bytes": sum(L["ext"]) * kvh * 4 + kept * kvh * (2 * 2 * VEC + 8 + 2 * 2 * HD),
                "flops": sum(L["ext"]) * kvh * 4}
    ext, T = [L["ext"][i] for i in L["of"]], sum(L["q"])
    if case["op"] == "attend":
        kv = L["q"] if case["local"] else [0] * len(L["q"])
        pairs = sum(q * (e + m) for q, e, m in zip(L["q"], ext, kv))
        return {"bytes": sum(L["ext"]) * kvh * 2 * VEC + sum(kv) * kvh * 2 * 2 * HD + T * h * (4 * HD + 4),
                "flops": pairs * h * 4 * HD}
    pairs = sum(q * e for q, e in zip(L["q"], ext))
    return {"bytes": sum(L["ext"]) * kvh * (VEC + 4) + T * h * (2 * HD + 4), "flops": pairs * h * 2 * HD}


# ------------------------------------------------------------------------------------------------ 64 bits
def _exact_vectors(x):
    """The cached form's values of fp16 vectors [..., 64], in 64 bits."""
    x = x.double()
    lo, hi = x.min(-1, keepdim=True)[0].clamp(max=0), x.max(-1, keepdim=True)[0].clamp(min=0)
    want = (hi - lo) / torch.full_like(lo, 15.0)
    unit = torch.exp2(torch.floor(torch.log2(want.clamp(min=2.0 ** -40)) + 2.0 ** -30) - 6).clamp(min=2.0 ** -20)
    step = torch.ceil(want / unit) * unit
    n = torch.where(step > 0, x / step, 0)
    z = torch.where(step > 0, -lo / step, 0).round().clamp(max=15)
    top = torch.where(step > 0, (65504.0 / step).floor(), 0)
    return ((torch.minimum(torch.maximum(n.round(), -top), top) + z).clamp(0, 15) - z) * step


def _exact_cached(b, par):
    """The values of packed vectors, by their bits."""
    word = b.contiguous().view(torch.int32)
    n = torch.arange(HD, device=b.device) % 8
    c = (word.repeat_interleave(8, -1) >> (4 * (n // 2) + 16 * (n % 2))) & 15
    return (c - (par & 15)[..., None]).double() * (par & ~15).view(torch.float16)[..., None].double()


def exact(case, seed):
    s = prepare(case, seed)
    L, kvh, group, h = _lens(case), s["kvh"], s["group"], s["heads"]
    if s["op"] == "append":
        kv = s["qkv"].view(-1, h + 2 * kvh, HD)
        return {"k": _exact_vectors(kv[:, h:h + kvh]).flatten(1), "v": _exact_vectors(kv[:, h + kvh:]).flatten(1)}
    if s["op"] == "evict":
        k, v, kept, mass = [], [], torch.full_like(s["kept"], -1), torch.zeros_like(s["d_mass"], dtype=torch.float64)
        for c, m in enumerate(L["ext"]):
            keep = min(case["keep"], m)
            recent = min(case["recent"], keep)
            w = s["mass"][c, :, :m - recent].double()
            # the most weight first, of equal ones the lowest index: by the pair (weight, -index), whole numbers here
            rank = w * 64 * 2 ** 20 - torch.arange(m - recent, device="cuda")
            best = rank.topk(keep - recent, -1)[1]
            at = torch.cat([best, torch.arange(m - recent, m, device="cuda").expand(kvh, -1)], 1).sort(-1)[0]
            kept[c, :, :keep], mass[c, :, :keep] = at.int(), s["mass"][c].double().gather(1, at)
            head = torch.arange(kvh, device="cuda")[:, None]
            k.append(_exact_cached(s["k4"][c][head, at], s["kp"][c][head, at]).transpose(0, 1).flatten(1))
            v.append(_exact_cached(s["v4"][c][head, at], s["vp"][c][head, at]).transpose(0, 1).flatten(1))
        return {"kept": kept, "mass": mass, "k": torch.cat(k), "v": torch.cat(v)}
    if work(case)["flops"] > 4e12:
        return None
    st = _starts(L["q"])
    o, lse = [], torch.empty(h, s["T"], dtype=torch.float64, device="cuda")
    mass = torch.zeros(len(L["ext"]), kvh, s["k4"].shape[2], dtype=torch.float64, device="cuda")
    for i, m in enumerate(L["q"]):
        c, e = L["of"][i], L["ext"][L["of"][i]]
        x = s["qkv"][st[i]:st[i] + m].double().view(m, h + 2 * kvh, HD).transpose(0, 1)
        out = torch.empty(h, m, HD, dtype=torch.float64, device="cuda") if s["op"] == "attend" else None
        for j in range(h):
            g = j // group
            key = _exact_cached(s["k4"][c, g, :e], s["kp"][c, g, :e])
            if s["op"] == "mass":
                mass[c, g, :e] += torch.exp(x[j] @ key.T / 8 - s["lse"][j, st[i]:st[i] + m, None].double()).sum(0)
                continue
            val = _exact_cached(s["v4"][c, g, :e], s["vp"][c, g, :e])
            if s["local"]:
                key, val = torch.cat([key, x[h + g]]), torch.cat([val, x[h + kvh + g]])
            y = x[j] @ key.T / 8
            lse[j, st[i]:st[i] + m] = torch.logsumexp(y, -1)
            out[j] = torch.softmax(y, -1) @ val
        if s["op"] == "attend":
            o.append(out.transpose(0, 1).flatten(1))
    return {"mass": mass} if s["op"] == "mass" else {"o": torch.cat(o), "lse": lse}
