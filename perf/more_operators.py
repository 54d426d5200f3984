"""The operators of a feed-forward layer over 8-bit rows and weights, as cases that
can be timed and compared: their plain form in elementary torch operations, and
the calls a user's program makes of phobos_amd.

A case names its "op" and sizes:
  norm     h = x + r; the root-mean-square norm of h times a gain, in 8 bits;
  glu      silu(gate) * up of rows [gate | up], in 8 bits;
  gemm     C = A @ W for A and W in 8 bits;
  grouped  the same for rows sorted by expert, each with its expert's W, and
           with or without a list of which of A's rows they are.

Both forms take the same bytes:
  rows     e4m3 codes [M, K] and a scale (f32) for every 128 of a row's K,
           [M, S], of which the first ceil(K / 128) count;
  weights  e4m3 codes [E, N, K] and a scale (f32) for every 128 x 128,
           [E, ceil(N / 128), ceil(K / 128)].
A code c stands for c * scale; the largest magnitude of a row's 128 (of a block of
weights) has the code 448 or -448.
"""
import math
import os
import sys

import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
WORKSPACE = 64 << 20  # bound to the stream once, as a serving program does
TYPES = {16: torch.float16, 32: torch.float32}
F8 = torch.float8_e4m3fn
EPS = 1e-5


def _norm(bits, M, K, residual, **kw):
    return dict(kw, op="norm", bits=bits, M=M, K=K, residual=residual)


def _glu(bits, M, K, **kw):
    return dict(kw, op="glu", bits=bits, M=M, K=K)


def _gemm(bits, M, N, K, **kw):
    return dict(kw, op="gemm", bits=bits, M=M, N=N, K=K)


def _grouped(bits, M, N, K, experts, idle, tokens, **kw):
    """M rows over `experts` groups, `idle` of them empty; of A's `tokens` rows by
    a list, or (tokens 0) in A's own order."""
    return dict(kw, op="grouped", bits=bits, M=M, N=N, K=K, experts=experts, idle=idle,
                tokens=tokens)


def listed():
    return [
        # one token of a decode step: the launch is most of it
        _norm(16, 1, 4096, True, name="norm_token"),
        # a batch of f32 rows before the first layer, nothing to add yet
        _norm(32, 1000, 4144, False, name="norm_f32_ragged"),
        # a prompt's rows with the layer's sum
        _norm(16, 16384, 8192, True, name="norm_prompt"),
        # the tokens of a served batch between the two products
        _glu(16, 32, 4096, name="glu_batch"),
        # a prompt's rows between the two products, no whole number of 128
        _glu(32, 4133, 5520, name="glu_f32_prompt"),
        # one token through a projection of the BASELINE GEMMs' width
        _gemm(16, 1, 4096, 4096, name="gemm_token"),
        # a served batch through a wide layer
        _gemm(16, 64, 16384, 8192, name="gemm_batch"),
        # a prompt of no round length, no extent a whole tile, f32 out
        _gemm(32, 1000, 1000, 4144, name="gemm_f32_ragged"),
        # a long prompt through a wide layer: the largest
        _gemm(16, 8192, 16384, 8192, name="gemm_prompt"),
        # eight tokens with two experts each: few rows each, most experts idle
        _grouped(16, 16, 2048, 4096, 32, 18, 8, name="experts_token"),
        # ragged groups in their own order, no extent a whole tile, f32 out
        _grouped(32, 1000, 1000, 1040, 7, 1, 0, name="experts_f32_ragged"),
        # a prompt's tokens, four experts each
        _grouped(16, 16384, 4096, 2048, 64, 3, 4096, name="experts_prompt"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "norm", "glu", "gemm", "gemm", "gemm", "grouped", "grouped"])
    bits = rng.choice([16, 16, 32])
    if op == "norm":
        K = 16 * _log(rng, 4, 1024)
        return _norm(bits, _log(rng, 1, min(16384, (1 << 26) // K)), K, rng.random() < 0.7)
    if op == "glu":
        K = 16 * _log(rng, 4, 512)
        return _glu(bits, _log(rng, 1, min(16384, (1 << 25) // K)), K)
    if op == "gemm":
        return _gemm(bits, _log(rng, 1, 8192), _log(rng, 64, 16384), 16 * _log(rng, 4, 512))
    experts = _log(rng, 4, 64)
    idle = rng.randrange(experts // 2)
    N, K = _log(rng, 64, 4096), 16 * _log(rng, 4, 128)
    M = max(experts - idle, _log(rng, 4, 16384))
    each = rng.choice([0, 1, 2, 4, 8])
    return _grouped(bits, M, N, K, experts, idle, -(-M // each) if each else 0)


# ---------------------------------------------------------------- 8 bits
def _e4m3(q):
    """q (f64) rounded to e4m3, ties to even: steps of an eighth of the power of
    two below, 2^-9 at the least."""
    step = torch.exp2(torch.floor(torch.log2(q.abs().clamp(min=2.0 ** -6))) - 3)
    return (q / step).round().mul_(step).to(F8)


def _largest(t):
    """The largest magnitude of each 128 of the last axis [..., ceil(K / 128), 1],
    and t [..., ceil(K / 128), 128], filled up with zeros."""
    K = t.shape[-1]
    t = torch.nn.functional.pad(t, (0, -K % 128)).unflatten(-1, (-1, 128))
    return t.abs().amax(-1, keepdim=True), t


def _codes(t):
    """The codes of rows t (f32) and their largest magnitudes (f64), in 64 bits:
    in 32 a quotient next to the middle of two codes may end on the wrong side."""
    K = t.shape[-1]
    a, blocks = _largest(t.double())
    q = blocks * 448 / torch.where(a > 0, a, torch.ones_like(a))
    return _e4m3(q).flatten(-2)[..., :K], a.squeeze(-1)


def _rows_of(x):
    codes, a = _codes(x)
    return codes.contiguous(), (a / 448).float()


def _weights_of(w):
    """Codes and scales of weights [E, N, K]."""
    E, N, K = w.shape
    b = torch.nn.functional.pad(w, (0, -K % 128, 0, -N % 128))
    b = b.view(E, b.shape[1] // 128, 128, b.shape[2] // 128, 128)
    a = b.abs().amax((2, 4), keepdim=True)
    codes = (b * (448 / a.clamp(min=1e-30))).clamp(-448, 448).to(F8)
    codes = codes.view(E, b.shape[1] * 128, -1)[:, :N, :K].contiguous()
    return codes, (a / 448).view(E, b.shape[1], b.shape[3])


def _row_values(codes, scales):
    s = scales[:, : -(-codes.shape[-1] // 128)]
    return codes.float() * s.repeat_interleave(128, -1)[:, : codes.shape[-1]]


def _weight_values(codes, scales):
    E, N, K = codes.shape
    s = scales.repeat_interleave(128, 1)[:, :N].repeat_interleave(128, 2)[:, :, :K]
    return codes.float() * s


# ---------------------------------------------------------------- inputs
def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _hidden(g, M, K):
    """Rows as between two layers: normal, some channels large in every row, and
    each row of a magnitude of its own."""
    channel = 1 + 15 * (torch.rand(K, generator=g, device="cuda") < 0.01)
    return _normal(g, M, K) * channel * (0.5 + torch.rand(M, 1, generator=g, device="cuda"))


def _starts(case, seed):
    """The experts' first rows: idle ones are empty, the others ragged."""
    g = torch.Generator().manual_seed(int(seed) + 1)
    E, M = case["experts"], case["M"]
    live = torch.randperm(E, generator=g)[: E - case["idle"]]
    share = torch.randn(live.numel(), generator=g).mul(0.5).exp()
    extra = M - live.numel()
    edge = (share.cumsum(0) / share.sum() * extra).long()
    edge[-1] = extra
    counts = torch.zeros(E, dtype=torch.int64)
    counts[live] = 1 + edge.diff(prepend=torch.zeros(1, dtype=torch.int64))
    return torch.cat([torch.zeros(1, dtype=torch.int64), counts.cumsum(0)])


def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    op, t, M, K = case["op"], TYPES[case["bits"]], case["M"], case["K"]
    if op == "norm":
        return {"x": _hidden(g, M, K).to(t),
                "r": _normal(g, M, K).to(t) if case["residual"] else None,
                "gain": (1 + 0.2 * _normal(g, K)).to(t)}
    if op == "glu":
        return {"u": (_normal(g, M, 2 * K) * (0.5 + torch.rand(M, 1, generator=g, device="cuda"))
                      ).to(t)}
    E = case.get("experts", 1)
    rows = case.get("tokens", 0) or M
    i = {}
    i["a"], i["sa"] = _rows_of(_hidden(g, rows, K))
    i["w"], i["sw"] = _weights_of(_normal(g, E, case["N"], K) / K ** 0.5)
    blocks = i["sa"].shape[1]
    i["sa"] = torch.nn.functional.pad(i["sa"], (0, -blocks % 4), value=math.nan)  # whole 16 bytes
    if op == "grouped":
        starts = _starts(case, seed)
        i["starts"] = starts.int().cuda()
        i["most"] = int(starts.diff().max())  # rows of one expert
        i["list"] = (torch.randperm(M, generator=g, device="cuda") % rows).int() \
            if case["tokens"] else None
    return i


def prepare(case, seed):
    state = dict(_inputs(case, seed), case=case)
    op, t, M, K = case["op"], TYPES[case["bits"]], case["M"], case["K"]
    if op in ("norm", "glu"):
        state["q"] = torch.empty(M, K, dtype=F8, device="cuda")
        state["sq"] = torch.empty(M, -(-K // 512) * 4, device="cuda")
        if op == "norm":
            state["h"] = torch.empty(M, K, dtype=t, device="cuda")
    else:
        state["out"] = torch.empty(M, case["N"], dtype=t, device="cuda")
    torch.cuda.synchronize()
    return state


# ---------------------------------------------------------------- one pass
_lib = None


def _phobos():
    """The framework, with a workspace bound to the default stream, on which
    torch works here too."""
    global _lib
    if _lib is None:
        path = os.path.join(ROOT, "phobos-lang_amd")
        if path not in sys.path:
            sys.path.insert(0, path)
        import phobos_amd
        phobos_amd.init(0)
        phobos_amd.bind_workspace(None, WORKSPACE)
        _lib = phobos_amd
    return _lib


def _own_descriptors(px, state):
    """The descriptors of the 8-bit rows and weights: a program keeps them."""
    if "descriptors" not in state:
        codes, scales = (state["q"], state["sq"]) if "q" in state else (state["a"], state["sa"])
        rows = px.F8Rows(codes.data_ptr(), scales.data_ptr(), codes.shape[0], codes.shape[1],
                         codes.stride(0), scales.stride(0))
        weights = None
        if "w" in state:
            w = state["w"]
            weights = px.F8Weights(w.data_ptr(), state["sw"].data_ptr(), *w.shape)
        state["descriptors"] = rows, weights
    return state["descriptors"]


def _scales(state):
    return state["sq"][:, : -(-state["case"]["K"] // 128)]


def _own_run(state):
    px, case, op = _phobos(), state["case"], state["case"]["op"]
    dtype = px.F16 if case["bits"] == 16 else px.F32
    rows, weights = _own_descriptors(px, state)
    if op == "norm":
        r, h = state["r"], state["h"]
        px.launch_norm_f8(None, dtype, state["x"].data_ptr(), r.data_ptr() if case["residual"] else 0,
                          state["gain"].data_ptr(), h.data_ptr() if case["residual"] else 0, 0, rows,
                          case["M"], case["K"], EPS)
        return (h, state["q"], _scales(state)) if case["residual"] else (state["q"], _scales(state))
    if op == "glu":
        px.launch_glu_f8(None, dtype, state["u"].data_ptr(), rows)
        return state["q"], _scales(state)
    if op == "gemm":
        px.launch_gemm_f8(None, rows, weights, dtype, state["out"].data_ptr())
        return state["out"]
    order = state["list"]
    px.launch_gemm_f8_grouped(None, rows, weights, state["starts"].data_ptr(),
                              order.data_ptr() if case["tokens"] else 0, case["M"], dtype,
                              state["out"].data_ptr())
    return state["out"]


def _plain_norm(state):
    x, r = state["x"].float(), state["r"]
    h = (x if r is None else x + r.float()).to(state["x"].dtype)
    f = h.float()
    factor = torch.rsqrt(f.square().mean(-1, keepdim=True) + EPS)
    codes, a = _codes(f * state["gain"].float())
    scales = (a.float() * factor) / 448
    return (codes, scales) if r is None else (h, codes, scales)


def _plain_glu(state):
    gate, up = state["u"].float().chunk(2, -1)
    codes, a = _codes(gate / (1 + torch.exp(-gate)) * up)
    return codes, a.float() / 448


def _plain_gemm(state):
    w = _weight_values(state["w"], state["sw"])[0]
    return (_row_values(state["a"], state["sa"]) @ w.t()).to(state["out"].dtype)


def _plain_grouped(state):
    case, starts, order = state["case"], state["starts"], state["list"]
    E, K = case["experts"], case["K"]
    a = _row_values(state["a"], state["sa"])
    if order is not None:
        a = a[order.long()]
    # each expert's rows at its place in a batch of the largest group's size
    row = torch.arange(case["M"], device="cuda")
    expert = torch.searchsorted(starts[1:].long(), row, right=True)
    slot = row - starts[expert]
    batch = torch.zeros(E, state["most"], K, device="cuda")
    batch[expert, slot] = a
    w = _weight_values(state["w"], state["sw"]).transpose(1, 2).contiguous()
    return torch.bmm(batch, w)[expert, slot].to(state["out"].dtype)


def run(state):
    op = state["case"]["op"]
    if own:
        return _own_run(state)
    if op == "norm":
        return _plain_norm(state)
    if op == "glu":
        return _plain_glu(state)
    return _plain_gemm(state) if op == "gemm" else _plain_grouped(state)


# ---------------------------------------------------------------- what a pass needs
def work(case):
    op, e, M, K = case["op"], case["bits"] // 8, case["M"], case["K"]
    blocks = -(-K // 128)
    if op == "norm":  # x, and with a residual r and h; the gain; codes and scales
        return {"bytes": M * K * (e * (3 if case["residual"] else 1) + 1) + e * K + 4 * M * blocks,
                "flops": 0}
    if op == "glu":
        return {"bytes": M * K * (2 * e + 1) + 4 * M * blocks, "flops": 0}
    N, rows = case["N"], case.get("tokens", 0) or M
    live = case.get("experts", 1) - case.get("idle", 0)
    weights = live * (N * K + 4 * -(-N // 128) * blocks)
    return {"bytes": weights + rows * (K + 4 * blocks) + e * M * N, "flops": 2 * M * N * K}


# ---------------------------------------------------------------- in 64 bits
def _exact_quotients(t):
    """What the codes of rows t (f64) are rounded from, and the largest magnitudes."""
    M, K = t.shape
    at = torch.arange(K, device="cuda") // 128
    a = torch.zeros(M, -(-K // 128), dtype=torch.float64, device="cuda")
    a.scatter_reduce_(1, at.expand(M, K), t.abs(), "amax")
    return t / a[:, at] * 448, a


def _exact_product(a, sa, w, sw):
    M, K = a.shape
    N = w.shape[0]
    k = torch.arange(K, device="cuda") // 128
    x = a.to(torch.float64) * sa.double()[:, k]
    y = torch.empty(M, N, dtype=torch.float64, device="cuda")
    for n0 in range(0, N, 4096):
        n = torch.arange(n0, min(N, n0 + 4096), device="cuda")
        v = w[n0:n0 + 4096].to(torch.float64) * sw.double()[n // 128][:, k]
        y[:, n0:n0 + 4096] = x @ v.t().contiguous()
    return y


def exact(case, seed):
    i, op = _inputs(case, seed), case["op"]
    if op == "norm":
        x = i["x"].double()
        h = x if i["r"] is None else x + i["r"].double()
        kept = h.to(i["x"].dtype).double()  # what is stored is what the norm reads
        q, a = _exact_quotients((kept * i["gain"].double()).float().double())
        s = a / torch.sqrt((kept * kept).sum(1, keepdim=True) / case["K"] + EPS) / 448
        return (q, s) if i["r"] is None else (h, q, s)
    if op == "glu":
        u = i["u"].double()
        gate, up = u[:, : case["K"]], u[:, case["K"]:]
        q, a = _exact_quotients(gate * torch.sigmoid(gate) * up)
        return q, a / 448
    if op == "gemm":
        return _exact_product(i["a"], i["sa"], i["w"][0], i["sw"][0])
    out = torch.empty(case["M"], case["N"], dtype=torch.float64, device="cuda")
    edges = i["starts"].tolist()
    for e, (b, end) in enumerate(zip(edges, edges[1:])):
        if end > b:
            rows = i["list"][b:end].long() if case["tokens"] else slice(b, end)
            out[b:end] = _exact_product(i["a"][rows], i["sa"][rows], i["w"][e], i["sw"][e])
    return out
