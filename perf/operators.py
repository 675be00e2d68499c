"""Cases and plain forms of the serving and training operators around attention:

``qk_norm_rope``            root-mean-square norm of every query and key head and the rotation by
                            position, one pass; with its gradient
``paged_kv_append``         a step's keys (normed, rotated) and values into a paged cache, its
                            queries normed and rotated in the same call
``paged_attention``         attention of a step's tokens - one, a chunk, or a tree of drafts - over
                            that cache

``run`` computes each in elementary torch operations, or, where ``own`` is set, through this
repository's package.
"""
import functools
import math
import os
import sys

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_EPS = 1e-6
_TABLE = 65536          # positions of the rotation table


def _case(name, op, dtype, batch, tokens, heads_q, heads_kv, dim, rotary, interleaved=False, ragged=False,
          length=0, page=0, slots_first=False, tree=False):
    """``length``: tokens the longest sequence already has in the cache; ``ragged``: sequences of
    different lengths and padded rows behind the shorter ones; ``slots_first``: cache stored as
    (page, slot, head, D) instead of (page, head, slot, D)."""
    c = dict(op=op, dtype=dtype, batch=batch, tokens=tokens, heads_q=heads_q, heads_kv=heads_kv, dim=dim,
             rotary=rotary, interleaved=interleaved, ragged=ragged, length=length, page=page,
             slots_first=slots_first, tree=tree)
    if name:
        c["name"] = name
    return c


def listed():
    return [
        # queries and keys of one step of 32 sequences in a model without a paged cache
        _case("norm rope step", "norm", "bf16", 32, 1, 32, 8, 128, 128),
        # prefill of four sequences, grouped-query heads
        _case("norm rope prefill", "norm", "bf16", 4, 4096, 32, 8, 128, 128),
        # odd sizes: part of the head rotated, neighbouring pairs, a head of 80
        _case("norm rope odd", "norm", "f16", 3, 1777, 10, 5, 80, 32, interleaved=True),
        # gradient of the prefill shape: a training step
        _case("norm rope grad", "norm_grad", "bf16", 4, 4096, 32, 8, 128, 128),
        # gradient in 32 bits, an odd number of tokens
        _case("norm rope grad f32", "norm_grad", "f32", 1, 777, 8, 8, 64, 64),
        # decode step of 64 sequences into pages of 16 tokens
        _case("append step", "append", "bf16", 64, 1, 32, 8, 128, 128, length=2048, page=16),
        # chunks of a prefill of different lengths, cache stored slot by slot
        _case("append chunk", "append", "bf16", 8, 2048, 32, 8, 128, 128, ragged=True, length=8192, page=64,
              slots_first=True),
        # one token of one sequence: latency
        _case("attention one", "attention", "f16", 1, 1, 32, 32, 128, 0, length=1024, page=16),
        # decode step of a batch at the size of the benchmark's decode workload, grouped heads
        _case("attention step", "attention", "bf16", 32, 1, 32, 8, 128, 0, ragged=True, length=8192, page=32),
        # a tree of 16 drafted tokens for each of 8 sequences
        _case("attention tree", "attention", "bf16", 8, 16, 32, 8, 128, 0, ragged=True, length=8192, page=16,
              tree=True),
        # odd sizes: seven drafts, pages of 24 tokens, heads of 64
        _case("attention tree odd", "attention", "f16", 5, 7, 12, 4, 64, 0, ragged=True, length=2500, page=24,
              slots_first=True, tree=True),
        # 64 drafts over long caches: as much tensor-core work as memory traffic
        _case("attention tree long", "attention", "bf16", 4, 64, 32, 8, 128, 0, ragged=True, length=32768, page=64,
              tree=True),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "norm_grad", "append", "attention", "attention"])
    heads_kv = rng.choice([1, 2, 4, 5, 8, 16])
    heads_q = heads_kv * rng.choice([1, 2, 3, 4, 8])
    if op in ("norm", "norm_grad"):
        dim = rng.choice([64, 80, 96, 128, 256])
        batch = _log(rng, 1, 32)
        most = max(1, 16384 * 40 * 128 // (batch * (heads_q + heads_kv) * dim))
        return _case(None, op, rng.choice(["bf16", "f16", "f32"]), batch, _log(rng, 1, min(8192, most)), heads_q,
                     heads_kv, dim, rng.choice([dim // 32 * 16, dim]), rng.random() < 0.3)
    dtype = rng.choice(["bf16", "bf16", "f16"])
    dim = rng.choice([64, 96, 128, 128])
    page = rng.choice([8, 16, 24, 32, 64, 128])
    batch = _log(rng, 1, 64)
    ragged, slots_first = rng.random() < 0.7, rng.random() < 0.5
    if op == "append":
        most = max(1, 16384 * 40 * 128 // (batch * (heads_q + heads_kv) * dim))
        length = _log(rng, 16, max(17, min(16384, (1 << 26) // (batch * heads_kv * dim))))
        return _case(None, op, dtype, batch, _log(rng, 1, min(2048, most)), heads_q, heads_kv, dim,
                     rng.choice([dim // 32 * 16, dim]), rng.random() < 0.3, ragged, length, page, slots_first)
    tokens = 1 if rng.random() < 0.4 else _log(rng, 2, 64)
    most = min((1 << 27) // (batch * heads_kv * dim), 32768 * 4 * 64 * 32 * 128 * 2 // 5 // (batch * heads_q * tokens * dim))
    return _case(None, op, dtype, batch, tokens, heads_q, heads_kv, dim, 0, False, ragged,
                 _log(rng, 16, max(17, min(65536, most))), page, slots_first, tokens > 1 and rng.random() < 0.8)


def _table(rotary, device):
    """cos, sin (positions, rotary / 2) in 32 bits, the angles taken in 64."""
    inv = 10000.0 ** (-torch.arange(0, rotary, 2, dtype=torch.float64, device=device) / rotary)
    angle = torch.arange(_TABLE, dtype=torch.float64, device=device)[:, None] * inv
    return angle.cos().float(), angle.sin().float()


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed))
    dt = _DTYPES[case["dtype"]]
    b, t, hq, hkv, d = (case[n] for n in ("batch", "tokens", "heads_q", "heads_kv", "dim"))

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, generator=g, device=dev) * scale).to(dt)

    s = {"case": dict(case)}
    # queries, keys and values as the fused projection leaves them: (B, T, heads, D) side by side
    qkv = normal(b, t, hq + 2 * hkv, d)
    s["q"], s["k"], s["v"] = (x.transpose(1, 2) for x in qkv.split([hq, hkv, hkv], dim=2))
    if case["op"] != "attention":
        s["cos"], s["sin"] = _table(case["rotary"], dev)
        s["q_weight"], s["k_weight"] = (1.0 + normal(d, scale=0.1).float()).to(dt), (1.0 + normal(d, scale=0.1).float()).to(dt)
    if case["op"] in ("norm", "norm_grad"):
        # every sequence at its own place: the last of the table's positions among them
        start = torch.randint(0, _TABLE - t + 1, (b, 1), generator=g, device=dev)
        start[0] = _TABLE - t
        s["positions"] = start + torch.arange(t, device=dev)
        if case["op"] == "norm_grad":
            s["dq"], s["dk"] = normal(b, hq, t, d), normal(b, hkv, t, d)
        return s

    length, page = case["length"], case["page"]
    lens = torch.full((b,), length, dtype=torch.int32, device=dev)
    new = torch.full((b,), t, dtype=torch.int32, device=dev)
    if case["ragged"]:
        lens = torch.randint(length // 4, length + 1, (b,), generator=g, device=dev, dtype=torch.int32)
        lens[-1] = length
        new = torch.randint((t + 1) // 2, t + 1, (b,), generator=g, device=dev, dtype=torch.int32)
        new[0] = t
    s["cache_lens"], s["new_lens"] = lens, new
    per_seq = -(-(length + t) // page)
    pages = b * per_seq + 7
    s["page_table"] = torch.randperm(pages, generator=g, device=dev)[:b * per_seq].reshape(b, per_seq).to(torch.int32)
    for name in ("k_cache", "v_cache"):
        shape = (pages, page, hkv, d) if case["slots_first"] else (pages, hkv, page, d)
        cache = torch.empty(shape, dtype=dt, device=dev)
        cache.normal_(generator=g)
        s[name] = cache.transpose(1, 2) if case["slots_first"] else cache
    if case["op"] == "attention" and case["tree"]:
        # drafted token j hangs from an earlier one; it sees its ancestors and itself
        parent = (torch.rand(b, t, generator=g, device=dev) * torch.arange(t, device=dev)).long()
        sees = torch.eye(t, dtype=torch.bool, device=dev).repeat(b, 1, 1)
        rows = torch.arange(b, device=dev)
        for j in range(1, t):
            sees[:, j] |= sees[rows, parent[:, j]]
        s["tree_mask"] = sees
    return s


# ---- plain forms ---------------------------------------------------------------------------

def _rotate(x, cos, sin, interleaved):
    """x (..., D) with cos, sin (..., R / 2): the first R values turned in pairs."""
    r = 2 * cos.shape[-1]
    turned, rest = x[..., :r], x[..., r:]
    if interleaved:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), dim=-1).flatten(-2)
    else:
        a, b = turned[..., :r // 2], turned[..., r // 2:]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)
    return torch.cat((turned, rest), dim=-1)


def _angles(s, positions):
    """cos and sin of (B, T) positions, one axis for the heads."""
    at = positions.long()
    return s["cos"][at][:, None], s["sin"][at][:, None]


def _norm_rope(x, weight, cos, sin, interleaved):
    x32 = x.float()
    n = x32 * torch.rsqrt(x32.square().mean(-1, keepdim=True) + _EPS) * weight.float()
    return _rotate(n, cos, sin, interleaved).to(x.dtype)


def _norm_rope_grad(dy, x, weight, cos, sin, interleaved):
    x32 = x.float()
    r = torch.rsqrt(x32.square().mean(-1, keepdim=True) + _EPS)
    n = x32 * r
    g = _rotate(dy.float(), cos, -sin, interleaved)
    dw = (g * n).sum((0, 1, 2), dtype=torch.float64)
    h = g * weight.float()
    dx = r * (h - n * (h * n).mean(-1, keepdim=True))
    return dx.to(x.dtype), dw.to(weight.dtype)


def _plain_append(s):
    c = s["case"]
    page = c["page"]
    step = torch.arange(c["tokens"], device=s["k"].device)
    at = s["cache_lens"].long()[:, None] + step
    real = step < s["new_lens"].long()[:, None]
    cos, sin = _angles(s, at)
    k = _norm_rope(s["k"], s["k_weight"], cos, sin, c["interleaved"])
    q = _norm_rope(s["q"], s["q_weight"], cos, sin, c["interleaved"])
    q = torch.where(real[:, None, :, None], q, torch.zeros_like(q))
    pages = s["page_table"].long().gather(1, at // page)
    return q, _put(s["k_cache"], pages, at % page, real, k), _put(s["v_cache"], pages, at % page, real, s["v"])


def _put(cache, pages, slots, real, new):
    """new (B, H, T, D) into the cache's slots; a padded token's slot keeps what it holds."""
    old = cache[pages, :, slots]
    cache[pages, :, slots] = torch.where(real[:, :, None, None], new.transpose(1, 2), old)
    return cache


def _visible(s, keys):
    """(B, T, keys): which slots of its sequence each token reads."""
    c = s["case"]
    t, dev = c["tokens"], s["q"].device
    lens, new = s["cache_lens"].long()[:, None, None], s["new_lens"].long()[:, None, None]
    draft = torch.arange(keys, device=dev) - lens                        # (B, 1, keys)
    inside = (draft >= 0) & (draft < new)
    j = draft.clamp(0, t - 1)
    if "tree_mask" in s:
        sees = s["tree_mask"].gather(2, j.expand(-1, t, -1))
    else:
        sees = j <= torch.arange(t, device=dev)[:, None]
    return (draft < 0) | (inside & sees)


def _plain_attention(s):
    c = s["case"]
    b, t, hq, hkv, d = (c[n] for n in ("batch", "tokens", "heads_q", "heads_kv", "dim"))
    table = s["page_table"].long()
    k, v = (s[n][table].transpose(1, 2).reshape(b, hkv, -1, d).float() for n in ("k_cache", "v_cache"))
    keys = k.shape[2]
    q = s["q"].reshape(b, hkv, hq // hkv * t, d).float()
    score = (q @ k.transpose(2, 3) * (1.0 / math.sqrt(d))).view(b, hq, t, keys)
    score.masked_fill_(~_visible(s, keys)[:, None], float("-inf"))
    p = torch.exp(score - score.amax(-1, keepdim=True))
    out = (p.view(b, hkv, -1, keys) @ v).view(b, hq, t, d) / p.sum(-1, keepdim=True)
    real = torch.arange(t, device=out.device) < s["new_lens"].long()[:, None]
    return torch.where(real[:, None, :, None], out, torch.zeros_like(out)).to(s["q"].dtype)


@functools.lru_cache(maxsize=1)
def _package():
    at = os.path.join(os.getcwd(), "cutile-python_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    import b200k
    return b200k


def run(state):
    s, c = state, state["case"]
    if own:
        b200k = _package()
        if c["op"] == "norm":
            return b200k.qk_norm_rope(s["q"], s["k"], s["q_weight"], s["k_weight"], s["cos"], s["sin"],
                                      s["positions"], eps=_EPS, interleaved=c["interleaved"])
        if c["op"] == "norm_grad":
            return b200k.qk_norm_rope_backward(s["dq"], s["dk"], s["q"], s["k"], s["q_weight"], s["k_weight"],
                                               s["cos"], s["sin"], s["positions"], eps=_EPS,
                                               interleaved=c["interleaved"])
        if c["op"] == "append":
            q = b200k.paged_kv_append(s["k"], s["v"], s["k_cache"], s["v_cache"], s["page_table"], s["cache_lens"],
                                      s["cos"], s["sin"], q=s["q"], q_weight=s["q_weight"], k_weight=s["k_weight"],
                                      new_lens=s["new_lens"], eps=_EPS, interleaved=c["interleaved"])
            return q, s["k_cache"], s["v_cache"]
        return b200k.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["page_table"], s["cache_lens"],
                                     new_lens=s["new_lens"], tree_mask=s.get("tree_mask"))
    if c["op"] == "norm":
        cos, sin = _angles(s, s["positions"])
        return (_norm_rope(s["q"], s["q_weight"], cos, sin, c["interleaved"]),
                _norm_rope(s["k"], s["k_weight"], cos, sin, c["interleaved"]))
    if c["op"] == "norm_grad":
        cos, sin = _angles(s, s["positions"])
        dq, dqw = _norm_rope_grad(s["dq"], s["q"], s["q_weight"], cos, sin, c["interleaved"])
        dk, dkw = _norm_rope_grad(s["dk"], s["k"], s["k_weight"], cos, sin, c["interleaved"])
        return dq, dk, dqw, dkw
    if c["op"] == "append":
        return _plain_append(s)
    return _plain_attention(s)


def work(case):
    b, t, hq, hkv, d = (case[n] for n in ("batch", "tokens", "heads_q", "heads_kv", "dim"))
    e = _DTYPES[case["dtype"]].itemsize
    if case["op"] in ("norm", "norm_grad"):
        moved = 2 if case["op"] == "norm" else 3
        n = b * t * (hq + hkv) * d
        return {"bytes": moved * n * e + b * t * (case["rotary"] * 4 + 8), "flops": (10 if moved == 2 else 20) * n}
    # lengths are drawn by prepare(): their means (5/8 of the longest, 3/4 of the step's tokens)
    live, new = (0.625 * case["length"], 0.75 * t) if case["ragged"] else (case["length"], t)
    if case["op"] == "append":
        n = b * new * (hq + 2 * hkv) * d
        return {"bytes": 2 * n * e + b * new * case["rotary"] * 4, "flops": 10 * n}
    keys = live + new
    return {"bytes": 2 * b * hkv * keys * d * e + 2 * b * hq * t * d * e, "flops": 4 * b * hq * new * keys * d}


# ---- from the definition, in 64 bits -------------------------------------------------------

def _exact_rope(x, weight, table_cos, table_sin, at, interleaved):
    """x (B, H, T, D) in 64 bits -> turned by a complex product; also the normed rows and 1 / rms."""
    x = x.double()
    rms = (x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + _EPS).sqrt()
    unit = x / rms
    turn = torch.complex(table_cos[at].double(), table_sin[at].double()).unsqueeze(1)
    y = unit * weight.double()
    return _turn(y, turn, interleaved), unit, rms


def _turn(y, turn, interleaved):
    r = 2 * turn.shape[-1]
    out = y.clone()
    first, second = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2), slice(r // 2, r))
    z = torch.complex(y[..., first].contiguous(), y[..., second].contiguous()) * turn
    out[..., first], out[..., second] = z.real, z.imag
    return out


def exact(case, seed):
    s = prepare(case, seed)
    inter = case["interleaved"]
    if case["op"] == "norm":
        return tuple(_exact_rope(s[n], s[n + "_weight"], s["cos"], s["sin"], s["positions"], inter)[0] for n in "qk")
    if case["op"] == "norm_grad":
        dx, dw = [], []
        for n in "qk":
            _, unit, rms = _exact_rope(s[n], s[n + "_weight"], s["cos"], s["sin"], s["positions"], inter)
            back = torch.complex(s["cos"][s["positions"]].double(), -s["sin"][s["positions"]].double()).unsqueeze(1)
            g = _turn(s["d" + n].double(), back, inter)
            dw.append((g * unit).flatten(0, 2).sum(0))
            h = g * s[n + "_weight"].double()
            along = (h * unit).sum(-1, keepdim=True) / unit.shape[-1]
            dx.append((h - along * unit) / rms)
        return dx[0], dx[1], dw[0], dw[1]
    lens, new = s["cache_lens"].tolist(), s["new_lens"].tolist()
    page, dev = case["page"], s["q"].device
    group = case["heads_q"] // case["heads_kv"]
    if case["op"] == "append":
        kc, vc = s["k_cache"].double(), s["v_cache"].double()
        at = torch.tensor(lens, device=dev)[:, None] + torch.arange(case["tokens"], device=dev)
        q = _exact_rope(s["q"], s["q_weight"], s["cos"], s["sin"], at, inter)[0]
        k = _exact_rope(s["k"], s["k_weight"], s["cos"], s["sin"], at, inter)[0]
        for b, n in enumerate(new):
            q[b, :, n:] = 0.0
            pages = s["page_table"][b].long()[at[b, :n] // page]
            kc[pages, :, at[b, :n] % page] = k[b, :, :n].transpose(0, 1)
            vc[pages, :, at[b, :n] % page] = s["v"][b, :, :n].transpose(0, 1).double()
        return q, kc, vc
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=dev)
    for b, (have, n) in enumerate(zip(lens, new)):
        where = torch.arange(have + n, device=dev)
        pages = s["page_table"][b].long()[where // page]
        hidden = torch.zeros(n, have + n, dtype=torch.bool, device=dev)
        sees = s["tree_mask"][b, :n, :n] if "tree_mask" in s else torch.ones(n, n, device=dev).tril().bool()
        hidden[:, have:] = ~sees
        for h in range(case["heads_kv"]):
            keys = s["k_cache"][pages, h, where % page].double()
            values = s["v_cache"][pages, h, where % page].double()
            for x in range(h * group, (h + 1) * group):
                score = s["q"][b, x, :n].double() @ keys.T / math.sqrt(case["dim"])
                out[b, x, :n] = torch.softmax(score.masked_fill(hidden, -math.inf), dim=-1) @ values
    return out
