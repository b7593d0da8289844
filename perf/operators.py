"""Decoding with rotated positions over a paged key-value cache: the cases that are timed, and their plain forms.

Four operators: the norm of queries and keys for each head with the position rotation in the same pass (forward, and
forward with backward), appending tokens to a paged cache, attention of one new token per sequence over its pages, and
eviction of a sequence's lightest rows down to a budget.  With ``own`` false, ``run`` computes them with elementary
torch operations in 32 bits (angles in 64); with ``own`` true it makes the calls a program makes of framework_amd.
"""
import math

import numpy as np
import torch

own = False

THETA, EPS = 10000.0, 1e-6
DEVICE = "cuda"


# ---- the cases -----------------------------------------------------------------------------------------------
def listed():
    return [
        # one new token of 8 sequences at far, unequal positions, 12 heads of 64: a launch's latency
        _rotate("rotate_tokens_8x12x64", batch=8, seq=1, q_heads=12, kv_heads=12, dim=64, rotary=64, start=100003, ragged=True),
        # a prompt of odd length in a grouped layout, half of each head rotated, neighbouring pairs
        _rotate("rotate_prompt_2047_32x128", batch=1, seq=2047, q_heads=32, kv_heads=8, dim=128, rotary=64, interleaved=True),
        # a short training batch with odd extents: forward and gradients
        _rotate("rotate_train_4x33_4x32", batch=4, seq=33, q_heads=4, kv_heads=4, dim=32, rotary=32, train=True),
        # a language model's training batch (8 sequences of 1024, 12 heads of 64): forward and gradients
        _rotate("rotate_train_8x1024_12x64", batch=8, seq=1024, q_heads=12, kv_heads=12, dim=64, rotary=64, train=True),
        # the first tokens of one answer: nothing but latency
        _step("step_1x12x64_57", seqs=1, q_heads=12, kv_heads=12, dim=64, page=16, longest=57, shortest=57),
        # the benchmark's decoding batch, 8 sequences of 32 heads of 128 behind 4096 positions, fp32 and int8 rows
        _step("step_8x32x128_4096", seqs=8, q_heads=32, kv_heads=32, dim=128, page=64, longest=4096, shortest=4096),
        _step("step_8x32x128_4096_int8", seqs=8, q_heads=32, kv_heads=32, dim=128, page=64, longest=4096, shortest=4096, int8=True),
        # requests of very unequal lengths in one batch, grouped heads, int8 rows, small pages
        _step("step_ragged_16x32g8_int8", seqs=16, q_heads=32, kv_heads=8, dim=128, page=16, longest=16385, shortest=3, int8=True),
        # one very long conversation, the cache's length the only axis to split; every position's weight is accumulated
        _step("step_long_131071_tracked", seqs=1, q_heads=32, kv_heads=8, dim=128, page=32, longest=131071, shortest=131071, tracked=True),
        # prompts of unequal lengths (a padded batch) taken into the cache as int8 rows, then the first token's attention
        _prompt("prompt_4x2047_int8", seqs=4, q_heads=12, kv_heads=12, dim=64, page=16, longest=2047, shortest=511, int8=True),
        # caches held to a budget while a prompt arrives in chunks
        _evict("evict_4x12x64_500", seqs=4, q_heads=12, kv_heads=12, dim=64, page=16, budget=500, chunk=77, recent=32),
        _evict("evict_8x32x128_4096", seqs=8, q_heads=32, kv_heads=32, dim=128, page=64, budget=4096, chunk=512, recent=256),
    ]


def _rotate(name, batch, seq, q_heads, kv_heads, dim, rotary, start=0, ragged=False, interleaved=False, train=False):
    return {"name": name, "op": "rotate", "batch": batch, "seq": seq, "q_heads": q_heads, "kv_heads": kv_heads, "dim": dim,
            "rotary": rotary, "start": start, "ragged": ragged, "interleaved": interleaved, "train": train}


def _step(name, seqs, q_heads, kv_heads, dim, page, longest, shortest, int8=False, tracked=False):
    return {"name": name, "op": "step", "seqs": seqs, "q_heads": q_heads, "kv_heads": kv_heads, "dim": dim, "page": page,
            "longest": longest, "shortest": shortest, "int8": int8, "tracked": tracked}


def _prompt(name, **kw):
    return dict(_step(name, **kw), op="prompt")


def _evict(name, seqs, q_heads, kv_heads, dim, page, budget, chunk, recent, int8=False):
    return {"name": name, "op": "evict", "seqs": seqs, "q_heads": q_heads, "kv_heads": kv_heads, "dim": dim, "page": page,
            "budget": budget, "chunk": chunk, "recent": recent, "int8": int8}


def draw(rng):
    def spread(lo, hi):
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    most = max(_cost(c) for c in listed())
    while True:
        kv = rng.choice([1, 2, 3, 4, 6, 8, 12, 16])
        group = rng.choice([1, 1, 2, 3, 4, 8])
        dim = rng.choice([32, 64, 64, 80, 96, 128, 128])
        page = rng.choice([8, 16, 32, 64, 128])
        op = rng.choice(["rotate", "train", "step", "step", "prompt", "evict"])
        heads = {"q_heads": kv * group, "kv_heads": kv, "dim": dim}
        if op in ("rotate", "train"):
            rotary = rng.choice([dim, dim, dim // 2])
            c = _rotate("", batch=spread(1, 32), seq=spread(1, 4096), rotary=rotary, start=rng.choice([0, 0, spread(1, 1 << 20)]),
                        ragged=rng.random() < 0.4, interleaved=rng.random() < 0.4, train=op == "train", **heads)
        elif op == "step":
            longest = spread(1, 100000)
            c = _step("", seqs=spread(1, 64), page=page, longest=longest, shortest=rng.choice([longest, spread(1, longest)]),
                      int8=dim % 16 == 0 and rng.random() < 0.5, tracked=rng.random() < 0.3, **heads)
        elif op == "prompt":
            longest = spread(1, 8192)
            c = _prompt("", seqs=spread(1, 16), page=page, longest=longest, shortest=rng.choice([longest, spread(1, longest)]),
                        int8=rng.random() < 0.5, **heads)
        else:
            budget = spread(16, 8192)
            c = _evict("", seqs=spread(1, 16), page=page, budget=budget, chunk=spread(1, 1024), recent=spread(1, budget), int8=rng.random() < 0.4, **heads)
        if _cost(c) <= most:
            del c["name"]
            return c


def _lengths(case):
    """From the shortest to the longest, evenly over the logarithm."""
    n, lo, hi = case["seqs"], case["shortest"], case["longest"]
    return [hi if n == 1 else int(round(lo * (hi / lo) ** (i / (n - 1)))) for i in range(n)]


def _row_bytes(case):
    return 2 * (case["dim"] + 4 if case["int8"] else 4 * case["dim"])


def work(case):
    d, hq, hk = case["dim"], case["q_heads"], case["kv_heads"]
    if case["op"] == "rotate":
        n = case["batch"] * case["seq"] * (hq + hk) * d
        return {"bytes": n * 4 * (4 if case["train"] else 2), "flops": n * (30 if case["train"] else 10)}
    n = case["seqs"]
    if case["op"] == "step":  # the new rows in, every row of the cache once, queries in, outputs out
        tokens, new = sum(_lengths(case)) + n, n
    elif case["op"] == "prompt":
        tokens = new = sum(_lengths(case))
    else:
        tokens, new = n * case["budget"], n * case["chunk"]
    by = tokens * hk * _row_bytes(case) + new * hk * (8 * d + _row_bytes(case)) + n * hq * d * 8
    if case["op"] == "evict":  # weights and positions of every row, and the protected rows that stand behind the budget
        by += n * hk * (case["budget"] + case["chunk"]) * 12 + 2 * n * hk * min(case["recent"], case["chunk"]) * _row_bytes(case)
    elif case["tracked"]:
        by += 8 * tokens * hk
    return {"bytes": by, "flops": 4 * tokens * hq * d}


def _cost(case):
    w = work(case)
    return w["bytes"] + w["flops"] / 50


# ---- inputs --------------------------------------------------------------------------------------------------
def _inputs(case, seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=g, device=DEVICE)

    d, hq, hk = case["dim"], case["q_heads"], case["kv_heads"]
    if case["op"] == "rotate":
        b, s = case["batch"], case["seq"]
        # one fused projection [B, S, Hq + 2 Hk, D]; the operator reads queries and keys where they lie in it
        s_in = {"qkv": normal(b, s, hq + 2 * hk, d), "gq": 1 + 0.2 * normal(d), "gk": 1 + 0.2 * normal(d)}
        if case["ragged"]:
            first = torch.randint(0, 4096, (b, 1), generator=g, device=DEVICE)
            s_in["positions"] = (first + torch.arange(s, device=DEVICE)).to(torch.int32)
        if case["train"]:
            s_in["dq"], s_in["dk"] = normal(b, hq, s, d), normal(b, hk, s, d)
        return s_in
    n = case["seqs"]
    s_in = {"q": 1.5 * normal(n, hq, 1, d)}
    if case["op"] == "evict":
        held, fresh = case["budget"], case["chunk"]
        s_in["w0"], s_in["w1"] = (_weights(normal(n, hk, m)) for m in (held, held + fresh))
    else:
        held, fresh = (max(_lengths(case)), 1) if case["op"] == "step" else (0, max(_lengths(case)))
    if held:
        s_in["k0"], s_in["v0"] = normal(n, hk, held, d), normal(n, hk, held, d)
    s_in["k"], s_in["v"] = normal(n, hk, fresh, d), normal(n, hk, fresh, d)
    return s_in


def _weights(z):
    """Accumulated attention: heavy-tailed, on a grid so that 32-bit sums are exact and ties occur."""
    return torch.clamp(torch.floor(torch.exp(1.5 * z) * 4096), max=2.0 ** 20) / 4096


def prepare(case, seed):
    s = {"case": case, **_inputs(case, seed)}
    if case["op"] == "rotate":
        b, t, hq, hk = case["batch"], case["seq"], case["q_heads"], case["kv_heads"]
        s["q"] = s["qkv"][:, :, :hq].permute(0, 2, 1, 3)
        s["k"] = s["qkv"][:, :, hq:hq + hk].permute(0, 2, 1, 3)
        if own:
            torch.cuda.synchronize()  # the framework's stream does not wait for torch's, which makes the inputs
        return s
    n, page = case["seqs"], case["page"]
    lens = {"step": lambda: _lengths(case), "prompt": lambda: [0] * n, "evict": lambda: [case["budget"]] * n}[case["op"]]()
    new = {"step": lambda: [1] * n, "prompt": lambda: _lengths(case), "evict": lambda: [case["chunk"]] * n}[case["op"]]()
    room = -(-max(a + b for a, b in zip(lens, new)) // page)
    s |= {"lens": lens, "new": new, "seen": list(lens), "room": room}
    (_own_cache if own else _plain_cache)(s)
    for name in ("k0", "v0", "w0"):
        s.pop(name, None)
    return s


def run(state):
    """One pass.  With ``own`` the outputs are unfinished work on the framework's stream, which torch's does not wait for, nor
    the other way round: wait for the whole device (torch.cuda.synchronize) before torch reads them, and again after it has
    read them before they are dropped or the next pass starts, since their memory goes back to an allocator at once."""
    op = state["case"]["op"]
    if op == "rotate":
        return _own_rotate(state) if own else _plain_rotate(state)
    return _own_serve(state) if own else _plain_serve(state)


# ---- plain forms ---------------------------------------------------------------------------------------------
def _angles(case, positions, seq):
    """cos and sin of every position's angles [B or 1, 1, S, R / 2], from 64-bit angles."""
    half = case["rotary"] // 2
    if positions is None:
        positions = torch.arange(seq, device=DEVICE)[None]
    at = (positions + case["start"]).double()
    a = at[:, None, :, None] * THETA ** (-torch.arange(half, device=DEVICE, dtype=torch.float64) / half)
    return torch.cos(a).float(), torch.sin(a).float()


def _pairs(case, x):
    r = case["rotary"]
    return (x[..., 0:r:2], x[..., 1:r:2]) if case["interleaved"] else (x[..., :r // 2], x[..., r // 2:r])


def _turn(case, x, cos, sin):
    lo, hi = _pairs(case, x)
    a, b = lo * cos - hi * sin, hi * cos + lo * sin
    turned = torch.stack([a, b], -1).flatten(-2) if case["interleaved"] else torch.cat([a, b], -1)
    return torch.cat([turned, x[..., case["rotary"]:]], -1)


def _plain_rotate(s):
    case = s["case"]
    cos, sin = _angles(case, s.get("positions"), case["seq"])
    out = []
    for x, g in ((s["q"], s["gq"]), (s["k"], s["gk"])):
        r = torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)
        out.append(_turn(case, x * r * g, cos, sin).contiguous())
    if case["train"]:
        for x, g, dy in ((s["q"], s["gq"], s["dq"]), (s["k"], s["gk"], s["dk"])):
            r = torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)
            dz = _turn(case, dy, cos, -sin)
            dn = dz * g
            out.append((r * dn - x * r ** 3 * (dn * x).mean(-1, keepdim=True)).contiguous())
            out.append((dz * x * r).sum((0, 1, 2)))
    return out


def _plain_cache(s):
    """Pages [pages, heads, page, D] in a shuffled order, a table of them per sequence, and what the cache holds already."""
    case, n, room = s["case"], s["case"]["seqs"], s["room"]
    shape = (n * room, case["kv_heads"], case["page"])
    g = torch.Generator(device=DEVICE)
    g.manual_seed(n * room)
    s["table"] = torch.randperm(n * room, generator=g, device=DEVICE).view(n, room)
    kind = torch.int8 if case["int8"] else torch.float32
    for name in ("kp", "vp"):
        s[name] = torch.zeros(shape + (case["dim"],), dtype=kind, device=DEVICE)
        s[name + "_scale"] = torch.zeros(shape, device=DEVICE) if case["int8"] else None
    for name, kind in (("weights", torch.float32), ("positions", torch.int32)):
        s[name] = torch.zeros((n, case["kv_heads"], room * case["page"]), dtype=kind, device=DEVICE)
    s["length"] = torch.tensor(s["lens"], device=DEVICE)
    s["fresh"] = torch.tensor(s["new"], device=DEVICE)
    s["seen_at"] = s["length"].clone()
    if "k0" in s:
        held = s["k0"].shape[2]
        _plain_append(s, s["k0"], s["v0"], torch.zeros_like(s["length"]), s["length"], torch.zeros_like(s["length"]))
        if "w0" in s:
            s["weights"][:, :, :held] = s["w0"]


def _quantized(x):
    """int8 codes and the row's scale: scale = max|x| / 127, codes rounded to nearest, halves away from zero."""
    scale = torch.clamp(x.abs().amax(-1) / 127.0, min=1e-8)
    y = x * (1.0 / scale)[..., None]
    whole = torch.trunc(y)
    codes = whole + torch.where((y - whole).abs() >= 0.5, torch.sign(y), torch.zeros_like(y))
    return torch.clamp(codes, -127, 127).to(torch.int8), scale


def _plain_append(s, k, v, length, count, seen):
    case, page = s["case"], s["case"]["page"]
    t = torch.arange(k.shape[2], device=DEVICE)
    seq, tok = torch.nonzero(t[None] < count[:, None], as_tuple=True)
    slot = length[seq] + tok
    where = (s["table"][seq, slot // page], slice(None), slot % page)
    for name, x in (("kp", k), ("vp", v)):
        rows = x[seq, :, tok]
        if case["int8"]:
            rows, scale = _quantized(rows)
            s[name + "_scale"][where] = scale
        s[name][where] = rows
    s["weights"][seq, :, slot] = 0.0
    s["positions"][seq, :, slot] = (seen[seq] + tok)[:, None].to(torch.int32)


def _plain_rows(s, name, slots):
    """The rows [n, heads, slots, D] of the first `slots` slots of every sequence, as the values they stand for."""
    case = s["case"]
    pages = -(-slots // case["page"])
    t = s["table"][:, :pages]
    x = s[name][t].transpose(1, 2).reshape(case["seqs"], case["kv_heads"], pages * case["page"], case["dim"])[:, :, :slots]
    if case["int8"]:
        scale = s[name + "_scale"][t].transpose(1, 2).reshape(case["seqs"], case["kv_heads"], pages * case["page"])[:, :, :slots]
        x = x.float() * scale[..., None]
    return x


def _plain_attend(s, length, slots, tracked):
    case, n = s["case"], s["case"]["seqs"]
    hk, d = case["kv_heads"], case["dim"]
    group = case["q_heads"] // hk
    k, v = _plain_rows(s, "kp", slots), _plain_rows(s, "vp", slots)
    q = s["q"].view(n, hk, group, d)
    behind = (torch.arange(slots, device=DEVICE)[None] >= length[:, None])[:, None, None]
    scores = (torch.matmul(q, k.transpose(-1, -2).contiguous()) * (d ** -0.5)).masked_fill(behind, float("-inf"))
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    if tracked:
        s["weights"][:, :, :slots] += p.sum(2)
    return torch.matmul(p, v).view(n, case["q_heads"], 1, d)


def _plain_evict(s):
    """The lightest rows leave; the rows behind the budget that stay take their slots, in slot order."""
    case, n, hk = s["case"], s["case"]["seqs"], s["case"]["kv_heads"]
    budget, slots = case["budget"], case["budget"] + case["chunk"]
    w, at = s["weights"][:, :, :slots], s["positions"][:, :, :slots].long()
    rank = torch.where(at >= (s["seen_at"] - case["recent"])[:, None, None], torch.full_like(w, float("inf")), w)
    order = torch.argsort(at, dim=-1)
    order = order.gather(-1, torch.argsort(rank.gather(-1, order), dim=-1, descending=True, stable=True))
    stays = torch.zeros_like(at, dtype=torch.bool).scatter_(-1, order[..., :budget], True)
    slot = torch.arange(slots, device=DEVICE)
    hole = ~stays[..., :budget]
    movers = torch.argsort((~(stays & (slot >= budget))).to(torch.int8), dim=-1, stable=True)
    movers = torch.nn.functional.pad(movers, (0, max(0, budget - slots)))
    source = torch.where(hole, movers.gather(-1, torch.clamp(hole.cumsum(-1) - 1, min=0)), slot[:budget])
    seq, head = torch.arange(n, device=DEVICE)[:, None, None], torch.arange(hk, device=DEVICE)[None, :, None]
    page, to = case["page"], slot[:budget].view(1, 1, -1)
    src, dst = (s["table"][seq, source // page], head, source % page), (s["table"][seq, to // page], head, to % page)
    for name in ("kp", "vp", "kp_scale", "vp_scale"):
        if s[name] is not None:
            s[name][dst] = s[name][src]
    for name in ("weights", "positions"):
        s[name][:, :, :budget] = s[name].gather(-1, source)


def _plain_serve(s):
    case = s["case"]
    _plain_append(s, s["k"], s["v"], s["length"], s["fresh"], s["seen_at"])
    if case["op"] == "evict":
        slots = case["budget"] + case["chunk"]
        s["weights"][:, :, :slots] += s["w1"]
        s["seen_at"] += case["chunk"]
        _plain_evict(s)
        out = _plain_attend(s, s["length"], case["budget"], False)
        return [out, s["weights"][:, :, :case["budget"]].clone(), s["positions"][:, :, :case["budget"]].clone()]
    slots = max(a + b for a, b in zip(s["lens"], s["new"]))
    out = [_plain_attend(s, s["length"] + s["fresh"], slots, case["tracked"])]
    if case["tracked"]:
        live = torch.arange(slots, device=DEVICE) < (s["length"] + s["fresh"])[:, None, None]
        out.append(torch.where(live, s["weights"][:, :, :slots], torch.zeros_like(s["weights"][:, :, :slots])))
    return out


# ---- the framework's calls -----------------------------------------------------------------------------------
class _OnDevice:
    """Device memory of the framework, for torch to look at; what it belongs to is freed when torch lets go of it."""

    def __init__(self, pointer, shape, kind, free):
        self.__cuda_array_interface__ = {"shape": tuple(shape), "typestr": kind, "data": (pointer, False), "version": 2}
        self.free = free

    def __del__(self):
        self.free()


def _seen_by_torch(tensor):
    pointer = _api().native.devPtr(tensor._id)
    return torch.as_tensor(_OnDevice(pointer, tensor.shape, "<f4", tensor.free), device=DEVICE)


def _ints_seen_by_torch(buffer, shape):
    native = _api().native
    return torch.as_tensor(_OnDevice(native.intBufferPtr(buffer), shape, "<i4", lambda: native.freeIntBuffer(buffer)), device=DEVICE)


def _api():
    if not hasattr(_api, "bound"):
        from framework_amd.api import bind
        from framework_amd.native import Native
        _api.bound = bind(Native())
    return _api.bound


def _given(x):
    """A tensor of the framework with the values of x."""
    import framework_amd
    t = _api().Tensor.zeros(list(x.shape))
    pointer = _api().native.devPtr(t._id)
    framework_amd.rocm().sync()
    torch.as_tensor(_OnDevice(pointer, x.shape, "<f4", lambda: None), device=DEVICE).copy_(x)
    torch.cuda.synchronize()
    return t


class _Held:
    """The framework's tensors and cache of one state; freed with the state."""

    def __init__(self):
        self.tensors, self.cache = [], None

    def __del__(self):
        for t in self.tensors:
            t.free()
        if self.cache is not None:
            self.cache.free()


def _own_cache(s):
    import framework_amd
    case, n = s["case"], s["case"]["seqs"]
    api, held = _api(), _Held()
    framework_amd.rocm().clear_cache()
    api.native.noGradStart()
    evicting = case["op"] == "evict"
    held.cache = api.PagedKvCache(n, s["room"] * case["page"], n * s["room"], case["page"], case["kv_heads"], case["dim"],
                                  quantized=case["int8"], tracked=evicting or case["tracked"])
    s["held"], s["seqs"] = held, [held.cache.add() for _ in range(n)]
    if "k0" in s:
        k0, v0 = _given(s["k0"]), _given(s["v0"])
        held.cache.append(s["seqs"], k0, v0, s["lens"])
        k0.free()
        v0.free()
    if "w0" in s:
        w0 = _given(s["w0"])
        held.cache.addWeights(s["seqs"], w0)
        w0.free()
    for name in ("q", "k", "v", "w1"):
        if name in s:
            s["own_" + name] = _given(s.pop(name))
            held.tensors.append(s["own_" + name])
    framework_amd.rocm().sync()


def _own_serve(s):
    case, cache, seqs = s["case"], s["held"].cache, s["seqs"]
    cache.append(seqs, s["own_k"], s["own_v"], s["new"] if case["op"] == "prompt" else None)
    scale = case["dim"] ** -0.5
    if case["op"] == "evict":
        cache.addWeights(seqs, s["own_w1"])
        cache.evict(seqs, case["budget"], case["recent"])
        out = cache.attend(seqs, s["own_q"], scale)
        weights, positions = cache.track(seqs)
        return [_seen_by_torch(out), _seen_by_torch(weights), _ints_seen_by_torch(positions, weights.shape)]
    out = [_seen_by_torch(cache.attend(seqs, s["own_q"], scale, accumulate=case["tracked"]))]
    if case["tracked"]:
        weights, positions = cache.track(seqs)
        _api().native.freeIntBuffer(positions)
        out.append(_seen_by_torch(weights))
    cache.truncate(seqs, s["lens"])
    return out


def _own_rotate(s):
    import framework_amd
    rocm, case, q, k = framework_amd.rocm(), s["case"], s["q"], s["k"]
    b, t, hq, hk, d = case["batch"], case["seq"], case["q_heads"], case["kv_heads"], case["dim"]
    positions = s.get("positions")
    out = [torch.empty((b, hq, t, d), device=DEVICE), torch.empty((b, hk, t, d), device=DEVICE)]
    plan = dict(batch=b, seq=t, head_dim=d, rotary_dims=case["rotary"], interleaved=case["interleaved"], theta=THETA, eps=EPS,
                offset=case["start"], positions=None if positions is None else positions.data_ptr(), position_stride=t)
    heads = [dict(x=x.data_ptr(), heads=h, strides=x.stride()[:3], gamma=g.data_ptr()) for x, h, g in ((q, hq, s["gq"]), (k, hk, s["gk"]))]
    rocm.qk_norm_rope(*[dict(h, out=y.data_ptr()) for h, y in zip(heads, out)], **plan)
    if case["train"]:
        grads = [torch.empty((b, hq, t, d), device=DEVICE), torch.empty(d, device=DEVICE),
                 torch.empty((b, hk, t, d), device=DEVICE), torch.empty(d, device=DEVICE)]
        rocm.qk_norm_rope_backward(*[dict(h, grad=dy.data_ptr(), dx=dx.data_ptr(), dgamma=dg.data_ptr())
                                     for h, dy, dx, dg in zip(heads, (s["dq"], s["dk"]), grads[0::2], grads[1::2])], **plan)
        out += grads
    return out


# ---- from the definition, in 64 bits -------------------------------------------------------------------------
def exact(case, seed):
    s = _inputs(case, seed)
    return _exact_rotate(case, s) if case["op"] == "rotate" else _exact_serve(case, s)


def _exact_rotate(case, s):
    b, t, hq, hk, d, rot = (case[x] for x in ("batch", "seq", "q_heads", "kv_heads", "dim", "rotary"))
    qkv = s["qkv"].double()
    at = s["positions"].double() if "positions" in s else torch.arange(t, device=DEVICE).double().expand(b, t)
    j = torch.arange(rot // 2, device=DEVICE)
    lo, hi = (2 * j, 2 * j + 1) if case["interleaved"] else (j, j + rot // 2)
    turn = torch.polar(torch.ones((b, t, 1, rot // 2), device=DEVICE, dtype=torch.float64),
                       ((at + case["start"])[..., None] * torch.exp(-math.log(THETA) * 2 * j.double() / rot))[:, :, None])
    ys, grads = [], []
    for first, h, g, dy in ((0, hq, s["gq"], s.get("dq")), (hq, hk, s["gk"], s.get("dk"))):
        x = qkv[:, :, first:first + h]
        inv = 1 / torch.sqrt((x * x).sum(-1, keepdim=True) / d + EPS)
        y = x * inv * g.double()
        z = torch.complex(y[..., lo], y[..., hi]) * turn
        y[..., lo], y[..., hi] = z.real, z.imag
        ys.append(y.transpose(1, 2))
        if dy is not None:
            dz = dy.double().transpose(1, 2).clone()
            z = torch.complex(dz[..., lo], dz[..., hi]) * turn.conj()
            dz[..., lo], dz[..., hi] = z.real, z.imag
            n = x * inv
            dn = dz * g.double()
            grads += [(inv * (dn - n * (dn * n).sum(-1, keepdim=True) / d)).transpose(1, 2), (dz * n).sum((0, 1, 2))]
    return ys + grads


def _exact_values(case, x):
    """What the cache's rows stand for."""
    if not case["int8"]:
        return x.double()
    scale = torch.maximum(x.abs().amax(-1, keepdim=True) / 127.0, torch.tensor(1e-8, device=DEVICE))
    y = (x * (1.0 / scale)).double()
    return torch.clamp(torch.sign(y) * torch.floor(y.abs() + 0.5), -127, 127) * scale.double()


def _exact_serve(case, s):
    n, hq, hk, d = (case[x] for x in ("seqs", "q_heads", "kv_heads", "dim"))
    outs, tracked, positions = [], [], []
    lengths = None if case["op"] == "evict" else _lengths(case)
    slots = None if lengths is None else max(lengths) + (case["op"] == "step")
    for i in range(n):
        if case["op"] == "step":
            rows = [torch.cat([s[a + "0"][i, :, :lengths[i]], s[a][i]], 1) for a in "kv"]
        elif case["op"] == "prompt":
            rows = [s[a][i, :, :lengths[i]] for a in "kv"]
        else:
            rows = [torch.cat([s[a + "0"][i], s[a][i]], 1) for a in "kv"]
            w = s["w1"][i].cpu().numpy().copy()
            w[:, :case["budget"]] += s["w0"][i].cpu().numpy()
            pick = torch.from_numpy(np.stack([_exact_pick(case, row) for row in w])).to(DEVICE)
            rows = [torch.gather(x, 1, pick[..., None].expand(hk, case["budget"], d)) for x in rows]
            tracked.append(torch.gather(torch.from_numpy(w).to(DEVICE), 1, pick).double())
            positions.append(pick.to(torch.int32))
        k, v = (_exact_values(case, x) for x in rows)
        q = s["q"][i].double().view(hk, hq // hk, d)
        p = torch.softmax((q @ k.transpose(1, 2).contiguous()) / math.sqrt(d), -1)
        outs.append((p @ v).reshape(hq, 1, d))
        if case.get("tracked"):
            tracked.append(torch.nn.functional.pad(p.sum(1), (0, slots - k.shape[1])))
    out = [torch.stack(outs)]
    if tracked:
        out.append(torch.stack(tracked))
    if positions:
        out.append(torch.stack(positions))
    return out


def _exact_pick(case, w):
    """Which row each slot of the budget holds afterwards: a row that stays keeps its slot, and the freed slots take the others in order."""
    slots, budget = len(w), case["budget"]
    protected = np.arange(slots) >= slots - case["recent"]
    best = np.lexsort((np.arange(slots), -w, ~protected))[:budget]
    pick = np.full(budget, -1)
    pick[best[best < budget]] = best[best < budget]
    pick[pick < 0] = np.sort(best[best >= budget])
    return pick
