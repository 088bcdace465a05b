"""Performance cases of the 4-bit products and of the selective-scan block's operators on one GPU.

Kinds of case (field "kind"):
  pack    rows to 4-bit codes with a shared power of two per 32 values, and back: what a program does
          that keeps weights (bf16) or activations (f32) in 4 bits; the result is the values kept.
  fp4     a product of 4-bit rows and 4-bit weights, the rows quantised within the pass.
  w4      a product of f32 rows and 4-bit weights.
  conv    the short causal convolution over the sequences of a batch, with the streams' stored inputs.
  scan    the selective state space scan over the same, with the streams' stored states.

Row counts and widths are those of the 0.6B FastConformer (d_model 1024, FF 4096, 1 to 14 frames per chunk, up
to 256 streams) and their multiples; the scan's widths are generic (an inner width of twice the model
width, 16 states per channel).
"""
import math
import os
import sys

import torch

own = False

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
F32, BF16 = 0, 1
TYPES = {"f32": (F32, torch.float32), "bf16": (BF16, torch.bfloat16)}
NONE, SILU, RELU, GLU = 0, 1, 2, 3
ALPHA = 0.5  # of the products that update a residual (a half step)


def listed():
    return [
        # the activations of one stream's 560 ms chunk
        {"name": "pack_chunk", "kind": "pack", "type": "f32", "rows": 7, "k": 1024},
        # a layer's weights at load
        {"name": "pack_weights", "kind": "pack", "type": "bf16", "rows": 8192, "k": 4096},
        # feed-forward up + SiLU of a 64-stream server's step
        {"name": "fp4_448_up", "kind": "fp4", "rows": 448, "n": 4096, "k": 1024, "act": SILU, "bias": False, "resid": False},
        # feed-forward down of a 256-stream server's step at the highest latency, the residual updated
        {"name": "fp4_3584_down", "kind": "fp4", "rows": 3584, "n": 4096, "k": 8192, "act": NONE, "bias": False, "resid": True},
        # one row through a wide matrix: a token or an 80 ms chunk
        {"name": "w4_1", "kind": "w4", "rows": 1, "n": 8192, "k": 2048, "act": NONE, "bias": True, "resid": False},
        # an odd number of rows, columns and inputs: a few streams, a head of odd width
        {"name": "w4_23_odd", "kind": "w4", "rows": 23, "n": 4099, "k": 1021, "act": NONE, "bias": True, "resid": False},
        # a prompt's gated projection
        {"name": "w4_1024_glu", "kind": "w4", "rows": 1024, "n": 4096, "k": 2048, "act": GLU, "bias": False, "resid": False},
        # one token of each of 64 streams
        {"name": "conv_step_64", "kind": "conv", "type": "f32", "streams": 64, "rows": 1, "ragged": False, "d": 2048, "taps": 4},
        # prompts of mixed lengths, some of them continued
        {"name": "conv_prompts", "kind": "conv", "type": "bf16", "streams": 24, "rows": 1500, "ragged": True, "d": 2048, "taps": 4},
        # one token of one stream: the smallest call
        {"name": "scan_step_1", "kind": "scan", "type": "f32", "streams": 1, "rows": 1, "ragged": False, "d": 2048, "n": 16,
         "groups": 1},
        # one long prompt: little width, a long axis
        {"name": "scan_prompt_8192", "kind": "scan", "type": "bf16", "streams": 1, "rows": 8192, "ragged": False, "d": 2048,
         "n": 16, "groups": 1},
        # prompts of mixed lengths, some of them continued
        {"name": "scan_prompts", "kind": "scan", "type": "f32", "streams": 12, "rows": 1000, "ragged": True, "d": 1536, "n": 16,
         "groups": 1},
    ]


def draw(rng):
    def log_int(lo, hi):
        return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))

    kind = rng.choice(["pack", "fp4", "fp4", "w4", "w4", "w4", "conv", "conv", "scan", "scan", "scan"])
    if kind == "pack":
        return {"kind": kind, "type": rng.choice(["f32", "bf16"]), "rows": log_int(1, 8192), "k": log_int(33, 4096)}
    if kind in ("fp4", "w4"):
        rows, k = log_int(1, 2048 if kind == "w4" else 3584), log_int(96, 8192 if rng.random() < 0.5 else 4096)
        n = log_int(64, 8192 if rows < 1024 else 4096)
        act = rng.choice([NONE, NONE, SILU, RELU, GLU])
        if rng.random() < 0.6:  # matrices are mostly of round sizes
            n, k = -(-n // 64) * 64, -(-k // 64) * 64
        return {"kind": kind, "rows": rows, "n": n + n % 2 if act == GLU else n, "k": k, "act": act,
                "bias": rng.random() < 0.5, "resid": act == NONE and rng.random() < 0.5}
    streams = log_int(1, 64)
    rows = 1 if rng.random() < 0.35 else log_int(2, max(2, 8192 // streams))
    case = {"kind": kind, "type": rng.choice(["f32", "bf16"]), "streams": streams, "rows": rows,
            "ragged": rows > 1 and rng.random() < 0.7, "d": log_int(100, 2048)}
    if rng.random() < 0.6:
        case["d"] = -(-case["d"] // 64) * 64
    if kind == "conv":
        return dict(case, taps=rng.choice([2, 3, 4, 4]))
    groups = rng.choice([1, 1, 2])
    return dict(case, d=case["d"] + case["d"] % groups, n=rng.choice([8, 16, 16, 11, 5]), groups=groups)


# ---- shapes ----------------------------------------------------------------------------------------


def lengths(case):
    """Rows of every sequence: all alike, or mixed with some empty ones."""
    n, rows = case["streams"], case["rows"]
    if not case["ragged"]:
        return [rows] * n
    return [0 if s % 7 == 4 else 1 + (rows - 1) * ((29 * s + 50) % 51) // 50 for s in range(n)]


def table(case):
    """A sequence's first row, its rows, the slot it goes on from (-1: from zero) and the slot it ends in; the
    slots written are others than those read, so that a pass can be made again."""
    out, first = [], 0
    for s, c in enumerate(lengths(case)):
        out.append((first, c, -1 if case["ragged"] and s % 3 == 1 else s, case["streams"] + s))
        first += c
    return out


def blocks(k):
    return -(-k // 32)


def padded(k):
    return -(-k // 128) * 128


def work(case):
    kind = case["kind"]
    if kind == "pack":
        m, k, size = case["rows"], case["k"], 4 if case["type"] == "f32" else 2
        return {"bytes": 2.0 * size * m * k + m * (k / 2 + blocks(k)), "flops": 2.0 * m * k}
    if kind in ("fp4", "w4"):
        m, n, k = case["rows"], case["n"], case["k"]
        nout = n // 2 if case["act"] == GLU else n
        return {"bytes": n * (k / 2 + blocks(k)) + 4.0 * m * k + 4.0 * m * nout * (2 if case["resid"] else 1) +
                (4.0 * n if case["bias"] else 0.0), "flops": 2.0 * m * n * k}
    m, d, size = sum(lengths(case)), case["d"], 4 if case["type"] == "f32" else 2
    slots = len(lengths(case)) + sum(t[2] >= 0 for t in table(case))
    if kind == "conv":
        return {"bytes": 2.0 * size * m * d + 4.0 * slots * (case["taps"] - 1) * d + 4.0 * d * (case["taps"] + 1),
                "flops": m * d * (2.0 * case["taps"] + 4)}
    n, g = case["n"], case["groups"]
    return {"bytes": size * m * (4.0 * d + 2 * g * n) + 4.0 * slots * d * n + 4.0 * d * (n + 2),
            "flops": m * d * (7.0 * n + 12)}


# ---- inputs ----------------------------------------------------------------------------------------


class _Rand:
    def __init__(self, seed, tag):
        self.g = torch.Generator(device="cuda").manual_seed(1000003 * tag + seed)

    def normal(self, *shape, std=1.0, mean=0.0):
        return torch.randn(*shape, generator=self.g, device="cuda") * std + mean

    def uniform(self, *shape):
        return torch.rand(*shape, generator=self.g, device="cuda")

    def ints(self, hi, *shape):
        return torch.randint(0, hi, shape, generator=self.g, device="cuda")


def _weights4(r, n, k):
    """Codes and scales of an n x k matrix as a checkpoint holds them: rows padded with zeros to 128 values."""
    kb, kp = blocks(k), padded(k)
    codes = r.ints(16, n, kp)
    codes[:, k:] = 0
    scales = torch.zeros(n, kp // 32, dtype=torch.int64, device="cuda")
    scales[:, :kb] = 124 - int(round(math.log2(k) / 2)) + r.ints(3, n, kb)
    return (codes[:, 0::2] | codes[:, 1::2] << 4).to(torch.uint8), scales.to(torch.uint8)


def prepare(case, seed):
    kind, dev = case["kind"], "cuda"
    st = {"case": case}
    if kind == "pack":
        m, k = case["rows"], case["k"]
        r, dt = _Rand(seed, 1), TYPES[case["type"]][1]
        st["x"] = (r.normal(m, k) * torch.exp(0.5 * r.normal(m, 1))).to(dt)
        st["q"] = torch.empty(m, padded(k) // 2, dtype=torch.uint8, device=dev)
        st["s"] = torch.empty(m, padded(k) // 32, dtype=torch.uint8, device=dev)
        st["out"] = torch.empty(m, k, dtype=dt, device=dev)
    elif kind in ("fp4", "w4"):
        m, n, k = case["rows"], case["n"], case["k"]
        r = _Rand(seed, 2)
        nout = n // 2 if case["act"] == GLU else n
        st["x"] = r.normal(m, -(-k // 4) * 4)  # rows of whole 16 bytes; the first k columns count
        st["wq"], st["ws"] = _weights4(r, n, k)
        st["bias"] = r.normal(n, std=0.1) if case["bias"] else None
        st["c0"] = r.normal(m, nout) if case["resid"] else None
        st["out"] = torch.empty(m, nout, device=dev)
        if kind == "fp4":
            st["q"] = torch.empty(m, padded(k) // 2, dtype=torch.uint8, device=dev)
            st["s"] = torch.empty(m, padded(k) // 32, dtype=torch.uint8, device=dev)
    else:
        seqs, d, dt = table(case), case["d"], TYPES[case["type"]][1]
        m, n = max(1, sum(t[1] for t in seqs)), len(seqs)
        r = _Rand(seed, 3)
        st["m"] = m
        st["seqs"] = torch.tensor(seqs, dtype=torch.int32, device=dev)
        st["xz"] = r.normal(m, 2 * d).to(dt)  # the block's input projection: x and the gate side by side
        st["out"] = torch.zeros(m, d, dtype=dt, device=dev)
        if kind == "conv":
            t = case["taps"]
            st["w"], st["bias"] = r.normal(d, t, std=1 / math.sqrt(t)), r.normal(d, std=0.1)
            st["state"] = r.normal(2 * n, t - 1, d)
        else:
            ns, g, rank = case["n"], case["groups"], 4 * -(-d // 64)
            st["u"] = r.normal(m, d).to(dt)
            st["dt"] = r.normal(m, d, std=0.5).to(dt)
            st["xdbc"], st["rank"] = r.normal(m, rank + 2 * g * ns).to(dt), rank  # the projection to dt's rank, B and C
            st["A"] = -(torch.arange(1, ns + 1, device=dev) * torch.exp(0.1 * r.normal(d, ns))).contiguous()
            st["skip"] = r.normal(d, std=0.2, mean=1.0)
            step = torch.exp(math.log(1e-3) + (math.log(0.1) - math.log(1e-3)) * r.uniform(d))
            st["dt_bias"] = torch.log(torch.expm1(step))  # softplus of it is a step of 0.001 to 0.1
            st["state"] = r.normal(2 * n, d, ns, std=0.5)
    return st


# ---- one pass --------------------------------------------------------------------------------------


def run(state):
    return _own(state) if own else _plain(state)


def _gpu():
    if not hasattr(_gpu, "g"):
        if os.path.join(REPO, "nemo-c_amd") not in sys.path:
            sys.path.insert(0, os.path.join(REPO, "nemo-c_amd"))
        import nemoasr
        _gpu.g, _gpu.api = nemoasr.Gpu(), nemoasr
    return _gpu.g, _gpu.api


def _own(st):
    g, api = _gpu()
    L, case, kind = api.lib(), st["case"], st["case"]["kind"]
    p = {k: v.data_ptr() if torch.is_tensor(v) else None for k, v in st.items()}
    g.begin()
    if kind == "pack":
        m, k, t = case["rows"], case["k"], TYPES[case["type"]][0]
        ldq, lds = padded(k) // 2, padded(k) // 32
        g.check(L.nk_fp4_quant(g.h, p["x"], t, k, p["q"], ldq, p["s"], lds, m, k))
        g.check(L.nk_fp4_dequant(g.h, p["q"], ldq, p["s"], lds, p["out"], t, k, m, k))
        g.end()
        return st["out"]
    if kind in ("fp4", "w4"):
        m, n, k = case["rows"], case["n"], case["k"]
        ldx, nout, ldq, lds = st["x"].shape[1], st["out"].shape[1], padded(k) // 2, padded(k) // 32
        resid = case["resid"]
        if resid:
            g.check(L.nk_copy(g.h, p["c0"], p["out"], m * nout))
        end = (p["wq"], ldq, p["ws"], lds, p["bias"], p["out"], nout, m, n, k, case["act"], int(resid), ALPHA if resid else 1.0)
        if kind == "fp4":
            g.check(L.nk_fp4_quant(g.h, p["x"], F32, ldx, p["q"], ldq, p["s"], lds, m, k))
            g.check(L.nk_gemm_fp4(g.h, p["q"], ldq, p["s"], lds, *end))
        else:
            g.check(L.nk_gemm_w4(g.h, p["x"], ldx, *end))
        g.end()
        return st["out"]
    d, t, n = case["d"], TYPES[case["type"]][0], case["streams"]
    size = st["xz"].element_size()
    if kind == "conv":
        g.check(L.nk_causal_conv(g.h, p["xz"], t, 2 * d, p["w"], p["bias"], p["state"], 2 * n, p["seqs"], n, case["rows"],
                                 p["out"], d, st["m"], d, case["taps"], SILU))
    else:
        ns, gr, rank = case["n"], case["groups"], st["rank"]
        b = p["xdbc"] + size * rank
        a = api.Scan(type=t, x=p["u"], ldx=d, dt=p["dt"], lddt=d, B=b, C=b + size * gr * ns, ldbc=rank + 2 * gr * ns,
                     z=p["xz"] + size * d, ldz=2 * d, y=p["out"], ldy=d, A=p["A"], skip=p["skip"], dt_bias=p["dt_bias"],
                     state=p["state"], slots=2 * n, seqs=p["seqs"], nseq=n, max_rows=case["rows"], M=st["m"], D=d, N=ns,
                     groups=gr, softplus=1)
        g.check(L.nk_ssm_scan(g.h, api.C.byref(a)))
    g.end()
    return {"y": st["out"], "state": st["state"][n:]}


# ---- the plain forms -------------------------------------------------------------------------------

VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _round4(x):
    """The values that rows keep in 4 bits: per 32 of them a power of two from the largest magnitude (64 bits: values
    lie next to the borders), to the nearest, ties to the even code."""
    m, k = x.shape
    v = torch.nn.functional.pad(x.double(), (0, padded(k) - k)).view(m, -1, 32)
    top = v.abs().amax(-1, keepdim=True)
    e = torch.clamp(torch.frexp(top)[1] - 3, min=-127)
    step = torch.exp2(e.double())
    a = (v / step).abs()
    code = ((a > 0.25).int() + (a >= 0.75).int() + (a > 1.25).int() + (a >= 1.75).int() + (a > 2.5).int() + (a >= 3.5).int() +
            (a > 5.0).int())
    kept = torch.tensor(VALUES, dtype=torch.float64, device=x.device)[code] * step * torch.sign(v)
    return torch.where(torch.isfinite(top), kept, math.nan).view(m, -1)[:, :k]


def _values4(q, s, k):
    """The values of codes (two to a byte, the low half first) and scales."""
    lut = torch.tensor(VALUES + tuple(-v for v in VALUES), device=q.device)
    codes = torch.stack((q & 15, q >> 4), -1).view(q.shape[0], -1).int()
    scale = torch.exp2(s.float() - 127).repeat_interleave(32, 1)
    return (lut[codes] * scale)[:, :k]


def _silu(v):
    return v / (1 + torch.exp(-v))


def _plain(st):
    case, kind = st["case"], st["case"]["kind"]
    if kind == "pack":
        return _round4(st["x"]).to(st["x"].dtype)
    if kind in ("fp4", "w4"):
        k, act = case["k"], case["act"]
        x = st["x"][:, :k]
        if kind == "fp4":
            x = _round4(x).float()
        y = x @ _values4(st["wq"], st["ws"], k).t()
        if st["bias"] is not None:
            y = y + st["bias"]
        if act == SILU:
            y = _silu(y)
        elif act == RELU:
            y = torch.clamp(y, min=0)
        elif act == GLU:
            a, b = y.chunk(2, 1)
            y = a / (1 + torch.exp(-b))
        return st["c0"] + ALPHA * y if case["resid"] else y
    return _plain_conv(st) if kind == "conv" else _plain_scan(st)


def _rows_of(st):
    """Per row its sequence and its place in it; per sequence its first row, rows and stored slot (-1: none)."""
    first, count, slot = (st["seqs"][:, i].long() for i in range(3))
    seq = torch.repeat_interleave(torch.arange(len(first), device=first.device), count, output_size=sum(lengths(st["case"])))
    return seq, torch.arange(len(seq), device=seq.device) - first[seq], first, count, slot


def _plain_conv(st):
    case = st["case"]
    d, t, n = case["d"], case["taps"], case["streams"]
    seq, place, first, count, slot = _rows_of(st)
    x = st["xz"][:len(seq), :d].float()
    before = torch.where((slot >= 0)[:, None, None], st["state"][slot.clamp(min=0)], 0.0)
    # the inputs of every sequence behind its stored ones, one sequence after another
    ends = torch.cumsum(count + t - 1, 0)
    start = ends - (count + t - 1)
    line = torch.empty(len(seq) + n * (t - 1), d, device=x.device)
    at = torch.arange(t - 1, device=x.device)
    line[(start[:, None] + at).view(-1)] = before.view(-1, d)
    line[start[seq] + t - 1 + place] = x
    window = line[(start[seq] + place)[:, None] + torch.arange(t, device=x.device)]
    y = _silu((window * st["w"].t()).sum(1) + st["bias"])
    out = torch.zeros(st["m"], d, device=x.device)
    out[:len(seq)] = y
    return {"y": out.to(st["out"].dtype), "state": line[((ends - (t - 1))[:, None] + at).view(-1)].view(n, t - 1, d)}


def _plain_scan(st):
    case = st["case"]
    d, ns, g, n = case["d"], case["n"], case["groups"], case["streams"]
    seq, place, first, count, slot = _rows_of(st)
    m = len(seq)
    u, xz, v = st["u"][:m].float(), st["xz"][:m].float(), st["dt"][:m].float() + st["dt_bias"]
    step = torch.clamp(v, min=0) + torch.log1p(torch.exp(-v.abs()))
    bc = st["xdbc"][:m, st["rank"]:].float().view(m, 2, g, ns).repeat_interleave(d // g, 2)
    before = torch.where((slot >= 0)[:, None, None], st["state"][slot.clamp(min=0)], 0.0)
    a = torch.exp(step[:, :, None] * st["A"])
    h = (step * u)[:, :, None] * bc[:, 0]
    begins = first[count > 0]
    h[begins] += a[begins] * before[count > 0]
    a[begins] = 0  # nothing crosses into a sequence
    reach = 1
    while reach < max(lengths(case), default=0):  # every row joined with those twice as far back each time
        h[reach:] += a[reach:] * h[:-reach].clone()
        a[reach:] *= a[:-reach].clone()
        reach *= 2
    y = (h * bc[:, 1]).sum(-1) + st["skip"] * u
    out = torch.zeros(st["m"], d, device=u.device)
    out[:m] = y * _silu(xz[:, d:])
    last = before.clone()
    last[count > 0] = h[(first + count - 1)[count > 0]]
    return {"y": out.to(st["out"].dtype), "state": last}


# ---- the same results in 64 bits -------------------------------------------------------------------


def _kept64(x):
    """Rows in 4 bits by distances: the nearest of the eight magnitudes, of two equally near the one at an even place."""
    m, k = x.shape
    out = torch.empty(m, k, dtype=torch.float64, device=x.device)
    mags = torch.tensor(VALUES, dtype=torch.float64, device=x.device)
    # what decides between two that are equally near
    favour = torch.tensor([0.0, 1e-18] * 4, dtype=torch.float64, device=x.device)
    for j in range(0, k, 32):
        b = x[:, j:j + 32].double()
        top = b.abs().amax(1)
        e = torch.floor(torch.log2(top))
        e = torch.where(torch.exp2(e) > top, e - 1, torch.where(torch.exp2(e + 1) <= top, e + 1, e))
        step = torch.exp2(torch.where(top > 0, e - 2, -127.0).clamp(min=-127.0))[:, None]
        dist = ((b / step).abs()[:, :, None] - mags).abs()
        near = dist.amin(-1, keepdim=True)
        at = torch.where(dist == near, favour, math.inf).argmin(-1)
        out[:, j:j + 32] = torch.copysign(mags[at] * step, b)
    return out


def exact(case, seed):
    kind = case["kind"]
    st = prepare(case, seed)
    if kind == "pack":
        return _kept64(st["x"])
    if kind in ("fp4", "w4"):
        k, act = case["k"], case["act"]
        x = _kept64(st["x"][:, :k]) if kind == "fp4" else st["x"][:, :k].double()
        n = case["n"]
        w = torch.empty(n, padded(k), dtype=torch.float64, device="cuda")
        for half in (0, 1):
            c = (st["wq"] >> (4 * half)) & 15
            low, e = (c & 1).double(), ((c >> 1) & 3).double()
            mag = torch.where(e == 0, low / 2, (1 + low / 2) * torch.exp2(e - 1))
            w[:, half::2] = torch.where(c >= 8, -mag, mag)
        w = (w.view(n, -1, 32) * torch.exp2(st["ws"].double() - 127)[:, :, None]).view(n, -1)[:, :k]
        y = x @ w.t() + (st["bias"].double() if case["bias"] else 0.0)
        if act == SILU:
            y = y * torch.sigmoid(y)
        elif act == RELU:
            y = torch.relu(y)
        elif act == GLU:
            y = y[:, :n // 2] * torch.sigmoid(y[:, n // 2:])
        return ALPHA * y + st["c0"].double() if case["resid"] else y
    out = torch.zeros(st["m"], case["d"], dtype=torch.float64, device="cuda")
    seqs, d, n = table(case), case["d"], case["streams"]
    old = [s[2] for s in seqs]
    state = torch.stack([st["state"][s].double() if s >= 0 else torch.zeros_like(st["state"][0]).double() for s in old])
    if kind == "conv":
        t, x = case["taps"], st["xz"][:, :d].double()
        for s, (first, count, _, _) in enumerate(seqs):
            line = torch.cat((state[s], x[first:first + count]))
            y = st["bias"].double() + sum(line[j:j + count] * st["w"][:, j].double() for j in range(t))
            out[first:first + count] = y * torch.sigmoid(y)
            state[s] = line[count:]
        return {"y": out, "state": state}
    ns, g = case["n"], case["groups"]
    u, step = st["u"].double(), torch.nn.functional.softplus(st["dt"].double() + st["dt_bias"].double(), threshold=100)
    bc = st["xdbc"][:, st["rank"]:].double().view(st["m"], 2, g, 1, ns)
    A, first = st["A"].double(), torch.tensor([s[0] for s in seqs], device="cuda")
    count = torch.tensor([s[1] for s in seqs], device="cuda")
    for i in range(max(s[1] for s in seqs)):
        live = (count > i).nonzero()[:, 0] if case["ragged"] else slice(None)
        row = first[live] + i
        b, c = ((bc[row, j].expand(-1, -1, d // g, -1)).reshape(-1, d, ns) for j in (0, 1))
        h = torch.exp(step[row][:, :, None] * A) * state[live] + (step[row] * u[row])[:, :, None] * b
        state[live] = h
        out[row] = (h * c).sum(-1)
    z = st["xz"][:, d:].double()
    return {"y": (out + st["skip"].double() * u) * z * torch.sigmoid(z), "state": state}
