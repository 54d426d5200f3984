"""The operators of a decode step over 4-bit weights and a 4-bit paged cache, as
cases that can be timed and compared: their plain form in elementary torch
operations, and the calls a user's program makes of phobos_amd.

A case names its "op" and sizes:
  gemv    y = x @ W for 1 .. 64 rows x, W [K, N] in 4-bit codes with a scale,
          and with or without a zero point, per group of K;
  attend  the queries of each sequence over its keys and values in the cache;
  store   a call's new tokens quantised into the cache's pages, and what they
          then stand for read back;
  pages   pages of the cache copied to other pages, in every layer.

Both forms take the same packed bytes:
  W       tiles of 16 columns by 128 rows, [N/16][K/128] of them, 1 KiB each:
          dword [q][r][j] (q, j < 4; r < 16) holds column 16T + r at k = 128b +
          32j + 8q + i, i = 0 .. 7, element i in nibble i/2 + 4 (i%2); padding
          is zero points.  Scales (f16) and zeros (u8) are [K/G, N].
  cache   pages of P tokens; for each head of a page P (D + 8) bytes: K's codes
          [P][D/2], two elements a byte, the even one in the low nibble; V's
          codes [P/4][D/8][4] dwords, token 4a + r, elements 8e .. 8e+7 from
          the low nibble on; then K's and V's [P] (f16 scale, f16 minimum).
          A code c stands for c * scale + minimum.
"""
import math
import os
import sys

import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
WORKSPACE = 64 << 20  # bound to the stream once, as a serving program does
TYPES = {16: torch.float16, 32: torch.float32}


def _gemv(bits, M, N, K, group, zeros, **kw):
    return dict(kw, op="gemv", bits=bits, M=M, N=N, K=K, group=group, zeros=zeros)


def _attend(bits, batch, heads, ratio, D, page, tokens, length, ragged, **kw):
    return dict(kw, op="attend", bits=bits, batch=batch, heads=heads, ratio=ratio, D=D, page=page,
                tokens=tokens, length=length, ragged=ragged)


def _store(bits, batch, heads, D, page, tokens, length, **kw):
    return dict(kw, op="store", bits=bits, batch=batch, heads=heads, D=D, page=page, tokens=tokens,
                length=length)


def _pages(layers, pages, copies, heads, D, page, **kw):
    return dict(kw, op="pages", layers=layers, pages=pages, copies=copies, heads=heads, D=D,
                page=page)


def listed():
    return [
        # one token through a small projection: the launch is most of it
        _gemv(16, 1, 1024, 1024, 32, False, name="w4_small"),
        # one token through a projection of the BASELINE GEMMs' width
        _gemv(16, 1, 4096, 4096, 128, True, name="w4_token"),
        # a few sequences' tokens in f32, no extent a whole tile or group
        _gemv(32, 5, 1000, 4136, 64, True, name="w4_f32_ragged"),
        # the largest batch through a wide layer
        _gemv(16, 64, 16384, 8192, 128, False, name="w4_batch"),
        # the first tokens of a single conversation, in f32, a head per query head
        _attend(32, 1, 4, 1, 64, 32, 1, 250, False, name="attend_start"),
        # a decode step of a served batch: grouped heads, every length its own
        _attend(16, 32, 8, 4, 128, 64, 1, 4096, True, name="attend_batch"),
        # one token over one very long document
        _attend(16, 1, 4, 8, 128, 128, 1, 100003, False, name="attend_long"),
        # a chunk of a prompt over what the cache holds of it, causal
        _attend(16, 2, 8, 4, 128, 64, 1000, 4133, False, name="attend_chunk"),
        # a decode step's new tokens into the cache
        _store(16, 32, 8, 128, 64, 1, 4096, name="store_token"),
        # a chunk of a prompt into the cache, in f32
        _store(32, 2, 8, 128, 64, 2000, 4133, name="store_chunk"),
        # the shared last pages of three forked sequences, in one layer
        _pages(1, 64, 3, 4, 64, 32, name="pages_fork"),
        # a compaction: many pages of every layer
        _pages(16, 512, 200, 8, 128, 64, name="pages_compact"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["gemv", "gemv", "gemv", "attend", "attend", "attend", "store", "pages"])
    if op == "gemv":
        return _gemv(rng.choice([16, 16, 32]), _log(rng, 1, 64), _log(rng, 64, 16384),
                     _log(rng, 32, 1024) * 8, rng.choice([32, 64, 128]), rng.random() < 0.5)
    D, page = rng.choice([64, 128]), rng.choice([32, 64, 128, 256])
    if op == "pages":
        pages = _log(rng, 16, 512)
        return _pages(_log(rng, 1, 16), pages, _log(rng, 1, max(2, pages * 2 // 5)),
                      rng.choice([1, 2, 4, 8]), D, rng.choice([32, 64]))
    heads, bits = rng.choice([1, 2, 4, 8, 16]), rng.choice([16, 16, 32])
    if op == "store":
        batch = _log(rng, 1, 64)
        tokens = 1 if rng.random() < 0.5 else _log(rng, 2, max(3, 4000 // batch))
        return _store(bits, batch, heads, D, page, tokens, tokens + _log(rng, 1, 2000))
    if rng.random() < 0.3:  # a chunk of a prompt
        batch, ratio = rng.choice([1, 2]), rng.choice([1, 2, 4])
        tokens = _log(rng, 2, 1000)
        return _attend(bits, batch, min(heads, 8), ratio, D, page, tokens,
                       tokens + _log(rng, 1, 3000), rng.random() < 0.5)
    batch, ratio = _log(rng, 1, 64), rng.choice([1, 2, 4, 5, 8, 16])
    most = min(131072, (1 << 20) // (batch * heads))  # keys of all heads, as in attend_batch
    return _attend(bits, batch, heads, ratio, D, page, 1, _log(rng, 1, most), rng.random() < 0.7)


# ---------------------------------------------------------------- packed bytes
def _pack_w4(codes):
    """codes u8 [K, N], padded to whole tiles, as the bytes of the tiles."""
    K, N = codes.shape
    c = codes.t().reshape(N // 16, 16, K // 128, 4, 4, 8).int()  # T r b j q i
    c = c.permute(0, 2, 4, 1, 3, 5)  # T b q r j i
    place = torch.tensor([4 * (i // 2 + 4 * (i % 2)) for i in range(8)], device=c.device)
    words = (c.long() << place).sum(-1)
    return torch.stack([(words >> s) & 255 for s in (0, 8, 16, 24)], -1).to(torch.uint8).flatten()


def _unpack_w4(packed, K, N):
    Kp, Np = -(-K // 128) * 128, -(-N // 16) * 16
    b = packed.view(Np // 16, Kp // 128, 4, 16, 4, 4)  # T b q r j byte
    c = torch.stack([b & 15, b >> 4], -1).flatten(-2)  # nibble 0 .. 7
    c = c.unflatten(-1, (2, 4)).transpose(-1, -2).flatten(-2)  # element 0 .. 7
    return c.permute(1, 4, 2, 5, 0, 3).reshape(Kp, Np)[:K, :N]  # b j q i, T r


def _quantise(x):
    """Codes, scale and minimum of rows x [..., D]: in 64 bits, as 32 put values
    next to the middle of two codes on the wrong side."""
    x = x.double()
    low, high = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    m = low.float().half().float()
    # by a tensor: by a number torch multiplies with its rounded reciprocal
    s = ((high - low) / torch.full_like(low, 15)).float().half().float().clamp(min=2.0 ** -24)
    return ((x - m) / s).round().clamp(0, 15).to(torch.uint8), s, m


def _param_bytes(s, m):
    return torch.cat([s, m], -1).half().contiguous().view(torch.uint8)  # [..., 4]


def _page_bytes(kc, ks, km, vc, vs, vm, P):
    """Whole pages from [B, L, H, ...] codes and parameters: [B, L/P, H, P (D + 8)] bytes."""
    B, L, H, D = kc.shape

    def paged(t):
        return t.view(B, L // P, P, H, -1).transpose(2, 3)  # B n H P ...

    k = paged(kc)
    k = (k[..., 0::2] | k[..., 1::2] << 4).flatten(3)
    v = paged(vc).unflatten(-1, (D // 8, 8)).unflatten(3, (P // 4, 4)).transpose(4, 5)
    v = (v[..., 0::2] | v[..., 1::2] << 4).flatten(3)
    return torch.cat([k, v, paged(_param_bytes(ks, km)).flatten(3),
                      paged(_param_bytes(vs, vm)).flatten(3)], -1)


def _cache_rows(pool, table, P, D):
    """K and V [B, H, L, D] in f32 that the pages of each sequence stand for."""
    t = pool[table.long().clamp(min=0)].transpose(1, 2)  # B H n bytes
    half = P * D // 2
    kc, vc, kp, vp = t.split([half, half, 4 * P, 4 * P], -1)
    kc = torch.stack([kc & 15, kc >> 4], -1).flatten(-2).unflatten(-1, (P, D))
    vc = torch.stack([vc & 15, vc >> 4], -1).flatten(-2).unflatten(-1, (P // 4, D // 8, 4, 8))
    vc = vc.transpose(-2, -3).reshape(kc.shape)
    kp = kp.contiguous().view(torch.float16).unflatten(-1, (P, 2)).float()
    vp = vp.contiguous().view(torch.float16).unflatten(-1, (P, 2)).float()
    k = kc.float() * kp[..., :1] + kp[..., 1:]
    v = vc.float() * vp[..., :1] + vp[..., 1:]
    return k.flatten(2, 3), v.flatten(2, 3)


# ---------------------------------------------------------------- inputs
def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _key_values(g, B, L, H, D):
    """Keys and values [B, L, H, D]: normal, some channels of the keys large, as
    after training, and each token of a magnitude of its own."""
    channel = 1 + 4 * (torch.rand(H, D, generator=g, device="cuda") < 0.05)
    token = 0.5 + torch.rand(B, L, 1, 1, generator=g, device="cuda")
    return _normal(g, B, L, H, D) * channel * token, _normal(g, B, L, H, D) * token


def _lengths(case, g):
    B, most = case["batch"], case["length"]
    lens = torch.full((B,), most, dtype=torch.int64, device="cuda")
    if case.get("ragged"):
        u = torch.rand(B, generator=g, device="cuda")
        lens = (case["tokens"] + u * (most - case["tokens"] + 1)).long().clamp(max=most)
        lens[0] = most
        if B >= 8:
            lens[B // 2] = 0  # a slot of the batch that holds no sequence now
    return lens


def _make_cache(case, g, lens):
    """The pool and table of sequences of these lengths; slots that hold no
    token, and pages that belong to nobody, are all ones (f16 NaN)."""
    B, H, D, P = case["batch"], case["heads"], case["D"], case["page"]
    n = -(-case["length"] // P)
    k, v = _key_values(g, B, n * P, H, D)
    blocks = _page_bytes(*_quantise(k), *_quantise(v), P)
    del k, v
    token = torch.arange(n * P, device="cuda").view(1, n, 1, P)
    empty = (token >= lens.view(B, 1, 1, 1)).expand(B, n, H, P)
    blocks[..., P * D:].view(B, n, H, 2, P, 4)[empty.unsqueeze(3).expand(B, n, H, 2, P)] = 255
    pages = B * n + 3
    order = torch.randperm(pages, generator=g, device="cuda")[: B * n].view(B, n)
    pool = torch.full((pages, H, P * (D + 8)), 255, dtype=torch.uint8, device="cuda")
    pool[order] = blocks
    held = torch.arange(n, device="cuda") * P < lens.view(B, 1)
    return pool, torch.where(held, order, -1).int()


def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    op, t = case["op"], TYPES.get(case.get("bits"))
    if op == "gemv":
        M, N, K, G = case["M"], case["N"], case["K"], case["group"]
        groups = -(-K // G)
        codes = (_normal(g, K, N) * 3 + 8).round().clamp(0, 15).to(torch.uint8)
        zeros = torch.randint(5, 11, (groups, N), generator=g, device="cuda").to(torch.uint8)
        scales = (0.5 + torch.rand(groups, N, generator=g, device="cuda")) / (3 * K ** 0.5)
        padded = torch.full((-(-K // 128) * 128, -(-N // 16) * 16), 8, dtype=torch.uint8,
                            device="cuda")
        padded[:K, :N] = codes
        return {"x": _normal(g, M, K).to(t), "w": _pack_w4(padded), "scales": scales.half(),
                "zeros": zeros if case["zeros"] else None}
    if op == "pages":
        layers, pages, n = case["layers"], case["pages"], case["copies"]
        words = case["heads"] * case["page"] * (case["D"] + 8) // 4
        pool = torch.randint(-2 ** 31, 2 ** 31, (layers, pages, words), generator=g, device="cuda",
                             dtype=torch.int32)
        order = torch.randperm(pages, generator=g, device="cuda")
        return {"pool": pool, "src": order[:n].cpu(), "dst": order[n:2 * n].cpu()}
    B, H, D, T = case["batch"], case["heads"], case["D"], case["tokens"]
    lens = _lengths(case, g)
    if op == "attend":
        pool, table = _make_cache(case, g, lens)
        q = _normal(g, B, T, H * case["ratio"], D).to(t)
        return {"q": q, "pool": pool, "table": table, "lens": lens.int()}
    n = -(-case["length"] // case["page"])
    table = torch.randperm(B * n + 3, generator=g, device="cuda")[: B * n].view(B, n).int()
    pool = torch.zeros(B * n + 3, H, case["page"] * (D + 8), dtype=torch.uint8, device="cuda")
    k, v = (x.to(t) for x in _key_values(g, B, T, H, D))
    return {"k": k, "v": v, "pool": pool, "table": table, "lens": lens.int()}


def prepare(case, seed):
    state = dict(_inputs(case, seed), case=case)
    op, t = case["op"], TYPES.get(case.get("bits"))
    if op == "gemv":
        state["out"] = torch.empty(case["M"], case["N"], dtype=t, device="cuda")
    elif op == "attend":
        state["out"] = torch.empty_like(state["q"])
    elif op == "store":
        state["out"] = torch.empty_like(state["k"]), torch.empty_like(state["v"])
    else:  # the lists of pages live on the host, where the pages are given out
        state["on_gpu"] = state["src"].cuda(), state["dst"].cuda()
        state["src"], state["dst"] = (state[k].int().numpy() for k in ("src", "dst"))
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


def _own_cache(px, state):
    """The descriptors of the cache and of the call's sequences: a program keeps them."""
    if "descriptors" not in state:
        case, pool, table = state["case"], state["pool"], state["table"]
        state["descriptors"] = (
            px.Kv4Cache(pool.data_ptr(), pool.shape[0], case["heads"], case["D"], case["page"]),
            px.Kv4Batch(table.data_ptr(), table.shape[1], state["lens"].data_ptr(), 0,
                        case["batch"], case["tokens"], case["length"],
                        case["batch"] * case["tokens"]))
    return state["descriptors"]


def _own_run(state):
    px, case, op = _phobos(), state["case"], state["case"]["op"]
    if op == "pages":
        pool = state["pool"]
        px.pages_copy(None, pool.data_ptr(), case["pages"], 4 * pool.shape[2], state["src"],
                      state["dst"], case["layers"], 4 * pool.stride(0))
        return pool
    dtype = px.F16 if case["bits"] == 16 else px.F32
    if op == "gemv":
        zeros = state["zeros"]
        px.launch_gemv_w4(None, dtype, state["x"].data_ptr(), state["w"].data_ptr(),
                          state["scales"].data_ptr(), zeros.data_ptr() if case["zeros"] else 0,
                          state["out"].data_ptr(), case["M"], case["N"], case["K"], case["group"],
                          1.0, 0.0)
        return state["out"]
    cache, batch = _own_cache(px, state)
    if op == "attend":
        px.launch_kv4_attention(None, cache, batch, dtype, state["q"].data_ptr(),
                                state["out"].data_ptr(), case["heads"] * case["ratio"],
                                case["D"] ** -0.5, True)
        return state["out"]
    k, v = state["out"]
    px.launch_kv4_append(None, cache, batch, dtype, state["k"].data_ptr(), state["v"].data_ptr())
    px.launch_kv4_read(None, cache, batch, dtype, k.data_ptr(), v.data_ptr())
    return k, v


def _plain_gemv(state):
    case, x = state["case"], state["x"]
    G = case["group"]
    q = _unpack_w4(state["w"], case["K"], case["N"]).float()
    g = torch.arange(case["K"], device="cuda") // G
    z = state["zeros"].float()[g] if case["zeros"] else 8.0
    return (x.float() @ ((q - z) * state["scales"].float()[g])).to(x.dtype)


def _plain_attend(state):
    case, q, lens = state["case"], state["q"], state["lens"]
    B, T, H, R, D = case["batch"], case["tokens"], case["heads"], case["ratio"], case["D"]
    k, v = _cache_rows(state["pool"], state["table"], case["page"], D)
    key = torch.arange(k.shape[2], device="cuda")
    row = lens.view(B, 1) - T + torch.arange(T, device="cuda")  # the rows' positions
    seen = key <= row.view(B, T, 1)  # B T L
    v = v.masked_fill((key >= lens.view(B, 1)).view(B, 1, -1, 1), 0)
    rows = q.float().view(B, T, H, R, D).permute(0, 2, 1, 3, 4).reshape(B, H, T * R, D)
    s = (rows @ k.transpose(-1, -2)) * D ** -0.5
    hidden = ~seen.view(B, 1, T, 1, -1).expand(B, H, T, R, -1).reshape(s.shape)
    s.masked_fill_(hidden, -math.inf)
    m = s.amax(-1, keepdim=True).clamp(min=-1e30)
    p = (s - m).exp_()
    o = (p @ v) / p.sum(-1, keepdim=True).clamp(min=1e-30)
    return o.view(B, H, T, R, D).permute(0, 2, 1, 3, 4).reshape(q.shape).to(q.dtype)


def _plain_store(state):
    case, pool = state["case"], state["pool"]
    B, T, H, D, P = case["batch"], case["tokens"], case["heads"], case["D"], case["page"]
    at = state["lens"].view(B, 1).long() - T + torch.arange(T, device="cuda")
    page = state["table"].long().gather(1, at // P).view(-1)
    slot = (at % P).view(-1)
    kc, ks, km = (x.view(B * T, H, -1) for x in _quantise(state["k"]))
    vc, vs, vm = (x.view(B * T, H, -1) for x in _quantise(state["v"]))
    half = P * D // 2
    head = torch.arange(H, device="cuda")
    kb = pool[..., :half].unflatten(-1, (P, D // 2))
    vb = pool[..., half:2 * half].unflatten(-1, (P // 4, D // 8, 4, 4))
    kp = pool[..., 2 * half:2 * half + 4 * P].unflatten(-1, (P, 4))
    vp = pool[..., 2 * half + 4 * P:].unflatten(-1, (P, 4))
    page, slot = page.view(-1, 1), slot.view(-1, 1)
    kb[page, head, slot] = kc[..., 0::2] | kc[..., 1::2] << 4
    vb[page, head, slot // 4, :, slot % 4] = (vc[..., 0::2] | vc[..., 1::2] << 4).unflatten(
        -1, (D // 8, 4))
    kp[page, head, slot] = _param_bytes(ks, km)
    vp[page, head, slot] = _param_bytes(vs, vm)
    # read back from the pages
    kr, vr = kb[page, head, slot], vb[page, head, slot // 4, :, slot % 4].flatten(-2)
    kr = torch.stack([kr & 15, kr >> 4], -1).flatten(-2).float()
    vr = torch.stack([vr & 15, vr >> 4], -1).flatten(-2).float()
    kq = kp[page, head, slot].view(torch.float16).float()
    vq = vp[page, head, slot].view(torch.float16).float()
    k, v = kr * kq[..., :1] + kq[..., 1:], vr * vq[..., :1] + vq[..., 1:]
    return k.view(B, T, H, D).to(state["k"].dtype), v.view(B, T, H, D).to(state["k"].dtype)


def run(state):
    op = state["case"]["op"]
    if own:
        return _own_run(state)
    if op == "gemv":
        return _plain_gemv(state)
    if op == "attend":
        return _plain_attend(state)
    if op == "store":
        return _plain_store(state)
    src, dst = state["on_gpu"]
    state["pool"][:, dst] = state["pool"][:, src]
    return state["pool"]


# ---------------------------------------------------------------- what a pass needs
def _keys(case):
    """Keys a pass reads of one head over all sequences: of ragged lengths the mean."""
    if not case["ragged"]:
        return case["batch"] * case["length"]
    B, mean = case["batch"], (case["tokens"] + case["length"]) / 2
    return case["length"] + (B - 1 - (B >= 8)) * mean


def work(case):
    op, e = case["op"], case.get("bits", 8) // 8
    if op == "gemv":
        M, N, K = case["M"], case["N"], case["K"]
        groups = -(-K // case["group"])
        return {"bytes": K * N / 2 + groups * N * (3 if case["zeros"] else 2) + e * M * (K + N),
                "flops": 2 * M * N * K}
    H, D = case["heads"], case["D"]
    if op == "pages":
        return {"bytes": 2 * case["copies"] * case["layers"] * H * case["page"] * (D + 8),
                "flops": 0}
    B, T = case["batch"], case["tokens"]
    if op == "store":  # the rows in, the pages out and in, the rows out
        return {"bytes": B * T * H * (2 * 2 * D * e + 2 * (D + 8)), "flops": 0}
    keys, Hq = _keys(case), H * case["ratio"]
    live = B - (case["ragged"] and B >= 8)
    pairs = T * keys - live * T * (T - 1) / 2  # row i of T sees all but the last T - 1 - i
    return {"bytes": keys * H * (D + 8) + 2 * B * T * Hq * D * e, "flops": 4 * pairs * Hq * D}


# ---------------------------------------------------------------- in 64 bits
def _exact_params(pool, page, head, at):
    """(scale, minimum) in f64 of pool bytes from `at` on."""
    b = [pool[page, head, at + i].long() for i in range(4)]
    pair = torch.stack([b[0] | b[1] << 8, b[2] | b[3] << 8], -1)
    pair = torch.where(pair >= 32768, pair - 65536, pair).short().view(torch.float16)
    return pair[..., 0].double(), pair[..., 1].double()


def _exact_row(pool, table, P, D, head, tokens):
    """K and V [tokens, D] in f64 of one head of one sequence, byte by byte."""
    page, slot = table.long()[tokens // P].view(-1, 1), (tokens % P).view(-1, 1)
    d = torch.arange(D, device="cuda")
    kb = pool[page, head, slot * (D // 2) + d // 2]
    vb = pool[page, head, P * D // 2 + ((slot // 4 * (D // 8) + d // 8) * 4 + slot % 4) * 4
              + d % 8 // 2]
    shift = (4 * (d % 2)).to(torch.uint8)
    ks, km = _exact_params(pool, page, head, P * D + 4 * slot)
    vs, vm = _exact_params(pool, page, head, P * D + 4 * P + 4 * slot)
    return ((kb >> shift) & 15).double() * ks + km, ((vb >> shift) & 15).double() * vs + vm


def _exact_stored(x):
    x = x.double()
    low, high = x.min(-1, keepdim=True).values, x.max(-1, keepdim=True).values
    m = low.float().half().double()
    s = ((high - low) / torch.full_like(low, 15)).float().half().double()
    s = torch.where(s < 2.0 ** -24, torch.full_like(s, 2.0 ** -24), s)
    return torch.clamp(torch.round((x - m) / s), 0, 15) * s + m


def exact(case, seed):
    op = case["op"]
    if op == "pages":
        return None  # bytes, not computed numbers
    i = _inputs(case, seed)
    if op == "store":
        return _exact_stored(i["k"]), _exact_stored(i["v"])
    if op == "gemv":
        M, N, K, G = case["M"], case["N"], case["K"], case["group"]
        k = torch.arange(K, device="cuda").view(-1, 1)
        y = torch.empty(M, N, dtype=torch.float64, device="cuda")
        for n0 in range(0, N, 2048):
            n = torch.arange(n0, min(N, n0 + 2048), device="cuda")
            element = k % 8
            word = (((n // 16 * -(-K // 128) + k // 128) * 4 + k % 32 // 8) * 16 + n % 16) * 4 \
                + k % 128 // 32
            nibble = element // 2 + 4 * (element % 2)
            byte = i["w"][word * 4 + nibble // 2]
            q = ((byte >> (4 * (nibble % 2)).to(torch.uint8)) & 15).double()
            z = i["zeros"][:, n].double()[k[:, 0] // G] if case["zeros"] else 8
            y[:, n0:n0 + 2048] = i["x"].double() @ (
                (q - z) * i["scales"][:, n].double()[k[:, 0] // G]).contiguous()
        return y
    q, out = i["q"].double(), torch.zeros_like(i["q"], dtype=torch.float64)
    T, R, D = case["tokens"], case["ratio"], case["D"]
    for b, n in enumerate(i["lens"].tolist()):
        if not n:
            continue
        tokens = torch.arange(n, device="cuda")
        hidden = tokens > (n - T + torch.arange(T, device="cuda")).view(T, 1, 1)
        for h in range(case["heads"]):
            k, v = _exact_row(i["pool"], i["table"][b], case["page"], D, h, tokens)
            rows = q[b, :, h * R:(h + 1) * R]  # T R D
            s = (rows.reshape(-1, D) @ k.t().contiguous()).view(T, R, n) / D ** 0.5
            p = torch.softmax(s.masked_fill(hidden, -math.inf), -1)
            o = (p.view(-1, n) @ v).view(T, R, D)
            out[b, :, h * R:(h + 1) * R] = o.nan_to_num(0.0) if T > n else o
    return out
