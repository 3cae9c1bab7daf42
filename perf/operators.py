"""Performance cases of the operators around a prefix cache whose observations differ in length.

A case names one call on a KvStore (bf16 pages [layer][observation][kv head][row][head_dim]):

  rope   qk_norm_rope_append: per-head norms of q and k, rotation at given positions, K / V into the pages
  cross  cross_attention: query tokens over each observation's own number of rows, with the rows' log-sum-exp
  mass   key_mass: the attention weight that every cached row got from the query tokens, accumulated
  evict  kv_evict: the heaviest rows of every page, moved into a smaller store

`run` computes a case in plain torch operations or, where `own` is true, through the package's entry points; `exact` computes it
from the definition in 64 bits.  Head layouts and prefix lengths are those of perf/cases.py; long caches, single tokens and
numbers of observations are what a deployment varies.
"""
import math

import torch

own = False

HEADS = {  # query heads, kv heads, head_dim
    "pi0": (8, 1, 256),
    "smolvla": (15, 5, 64),
    "lm": (20, 5, 128),
}


def listed():
    return [
        # one token of one robot's dialogue, far into a context stretched eightfold: a launch's latency
        {"name": "rope_step", "kind": "rope", "heads": "lm", "obs": 1, "tokens": 1, "ragged": False, "rot": 128, "interleaved": False,
         "scaling": "yarn", "factor": 8.0, "pos0": 100003, "f32": False},
        # the action tokens of a batch of robots, a part of each head rotated in pairs of neighbours, float32 projections
        {"name": "rope_chunk", "kind": "rope", "heads": "smolvla", "obs": 64, "tokens": 51, "ragged": False, "rot": 32,
         "interleaved": True, "scaling": "none", "factor": 1.0, "pos0": 241, "f32": True},
        # a backbone's prefix of images and text for parallel environments, padded to the longest
        {"name": "rope_prefix", "kind": "rope", "heads": "pi0", "obs": 33, "tokens": 816, "ragged": True, "rot": 256,
         "interleaved": False, "scaling": "linear", "factor": 4.0, "pos0": 0, "f32": False},
        # one token over one long cache: every row is read once
        {"name": "cross_step", "kind": "cross", "heads": "pi0", "obs": 1, "tokens": 1, "rows": 16001, "least": 16001, "pad": 0,
         "idle": False},
        # cross-attention layers of an action expert: prefixes of one to three views, padded language slots, one robot idle
        {"name": "cross_chunk", "kind": "cross", "heads": "smolvla", "obs": 64, "tokens": 50, "rows": 241, "least": 113, "pad": 17,
         "idle": True},
        # a suffix over prefixes of one to three views with wide heads
        {"name": "cross_suffix", "kind": "cross", "heads": "pi0", "obs": 64, "tokens": 51, "rows": 816, "least": 304, "pad": 0,
         "idle": False},
        # a whole prompt over long encoder states
        {"name": "cross_long", "kind": "cross", "heads": "lm", "obs": 4, "tokens": 816, "rows": 8190, "least": 4097, "pad": 0,
         "idle": False},
        # the weights of one token over a long cache
        {"name": "mass_step", "kind": "mass", "heads": "lm", "obs": 1, "tokens": 1, "rows": 16001, "least": 16001, "pad": 0, "idle": False},
        # what the action tokens of a batch looked at
        {"name": "mass_suffix", "kind": "mass", "heads": "pi0", "obs": 64, "tokens": 51, "rows": 816, "least": 304, "pad": 0,
         "idle": False},
        # what a prompt looked at in long encoder states
        {"name": "mass_long", "kind": "mass", "heads": "lm", "obs": 4, "tokens": 816, "rows": 8190, "least": 4097, "pad": 0, "idle": False},
        # one robot's prefix cut to half before its denoise loop
        {"name": "evict_one", "kind": "evict", "heads": "smolvla", "layers": 16, "obs": 1, "rows": 241, "least": 241, "keep": 120,
         "sink": 1, "recent": 49},
        # the prefixes of parallel environments cut to a common length, shorter ones among them
        {"name": "evict_batch", "kind": "evict", "heads": "pi0", "layers": 18, "obs": 64, "rows": 816, "least": 304, "keep": 387,
         "sink": 4, "recent": 48},
    ]


def _log_int(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    kind = rng.choice(["rope", "cross", "mass", "evict"])
    heads = rng.choice(sorted(HEADS))
    n_q, n_kv, hd = HEADS[heads]
    obs = _log_int(rng, 1, 64)
    if kind == "rope":
        f32 = rng.random() < 0.4
        most = 2.2e8 / (obs * (n_q + 2 * n_kv) * hd * (6 if f32 else 4))  # a drawn case costs no more than the largest listed one
        tokens = _log_int(rng, 1, max(1, min(816, int(most))))
        return {"kind": kind, "heads": heads, "obs": obs, "tokens": tokens, "ragged": rng.random() < 0.5,
                "rot": 2 * rng.randint(1, hd // 2) if rng.random() < 0.5 else hd // rng.choice([1, 2, 4]),
                "interleaved": rng.random() < 0.5, "scaling": rng.choice(["none", "linear", "ntk", "yarn"]),
                "factor": rng.choice([2.0, 4.0, 16.0]), "pos0": _log_int(rng, 1, 1000000), "f32": f32}
    if kind == "evict":
        rows = _log_int(rng, 16, 816)
        keep = rng.randint(1, rows)
        sink = rng.randint(0, min(keep, 8))
        layers = rng.randint(1, max(1, min(18, int(9e8 / (obs * keep * n_kv * hd * 8)))))
        return {"kind": kind, "heads": heads, "layers": layers, "obs": obs, "rows": rows, "least": rng.randint(0, rows),
                "keep": keep, "sink": sink, "recent": rng.randint(0, min(keep - sink, 48))}
    tokens = _log_int(rng, 1, max(1, min(816, int(1e8 / (obs * n_q * hd * 4)))))
    most = 2.0e11 / (obs * n_q * tokens * 4 * hd)
    rows = _log_int(rng, 1, max(2, min(16384, int(most), int(1e8 / (obs * n_kv * hd * 4)))))
    return {"kind": kind, "heads": heads, "obs": obs, "tokens": tokens, "rows": rows, "least": rng.randint(0, rows),
            "pad": rng.choice([0, 0, rng.randint(1, 48)]), "idle": rng.random() < 0.3}


# ------------------------------------------------------------------------------------------------- sizes
def _lens(case):
    """Rows (or tokens) of every observation, spread evenly from the fewest to the most."""
    n = case["obs"]
    hi = case["rows"] if "rows" in case else case["tokens"]
    lo = case["least"] if "least" in case else (hi * 3 // 8 if case["ragged"] else hi)
    lens = [hi - (hi - lo) * b // max(n - 1, 1) for b in range(n)]
    if case.get("idle") and n > 1:
        lens[n // 2] = 0
    return lens


def _pad_of(case, n):
    """The hidden rows of an observation of n rows: unused language slots in front of its last row."""
    hi = max(n - 1, 0)
    return max(hi - case["pad"], 0), hi


def _seen(case):
    return [n - (_pad_of(case, n)[1] - _pad_of(case, n)[0] if case["pad"] else 0) for n in _lens(case)]


# ------------------------------------------------------------------------------------------------- inputs
def _store(state, layers, obs, n_kv, hd, rows):
    """Pages of `rows` rows, random as a filled cache holds them; a KvStore around them where the package runs."""
    shape = (layers, obs, n_kv, rows, hd)
    if own:
        import vla_cpp_b200 as vb

        st = vb.KvStore(layers, obs, n_kv, hd, rows, 0)
        state["store"], k, v = st, st.k, st.v
    else:
        k = torch.empty(shape, dtype=torch.bfloat16, device="cuda")
        v = torch.empty_like(k)
    state["k"], state["v"] = k, v


def _plan(case, state):
    hd = HEADS[case["heads"]][2]
    f, m = _frequencies(case["rot"], case["scaling"], case["factor"])
    if own:
        import vla_cpp_b200 as vb

        state["freqs"], state["mscale"] = vb.rope_freqs(case["rot"], 10000.0, case["scaling"], case["factor"], 8192)
    else:
        state["freqs"], state["mscale"] = torch.tensor(f, dtype=torch.float64, device="cuda"), m
    assert case["rot"] <= hd


def _frequencies(rot, scaling, factor, base=10000.0, original=8192):
    """Angle per position of every rotated pair, and the factor on cos and sin."""
    if scaling == "ntk" and rot > 2:
        base = base * factor ** (rot / (rot - 2))
    f = [base ** (-2.0 * i / rot) for i in range(rot // 2)]
    if scaling == "linear":
        return [x / factor for x in f], 1.0
    if scaling != "yarn":
        return f, 1.0

    def pair_with_turns(turns):  # the (fractional) pair that turns this often within the original length
        return rot * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base))

    lo, hi = max(math.floor(pair_with_turns(32.0)), 0), min(math.ceil(pair_with_turns(1.0)), rot - 1)
    out = []
    for i, x in enumerate(f):
        ramp = min(max((i - lo) / max(hi - lo, 1e-3), 0.0), 1.0)
        out.append(x / factor * ramp + x * (1.0 - ramp))
    return out, 0.1 * math.log(factor) + 1.0


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def normal(*shape, std=1.0, dtype=torch.float32):
        return torch.empty(shape, dtype=dtype, device="cuda").normal_(0.0, std, generator=g)

    n_q, n_kv, hd = HEADS[case["heads"]]
    obs = case["obs"]
    order = torch.randperm(obs, generator=g, device="cuda")
    state = {"case": case, "lens": torch.tensor(_lens(case), dtype=torch.int32, device="cuda")[order].contiguous()}
    if case["kind"] == "rope":
        S = case["tokens"]
        # the projection's rows; every fourth column of a head is larger, as trained projections have it
        x = normal(obs * S, (n_q + 2 * n_kv) * hd)
        x.view(obs * S, -1, 4)[..., 1] *= 3.0
        state["x"] = x if case["f32"] else x.bfloat16()
        state["q_w"] = 1.0 + normal(hd, std=0.1)
        state["k_w"] = 1.0 + normal(hd, std=0.1)
        first = torch.randint(0, case["pos0"] + 1, (obs, 1), generator=g, device="cuda", dtype=torch.int32)
        state["pos"] = (first + torch.arange(S, device="cuda", dtype=torch.int32)).contiguous()
        state["row0"] = torch.randint(0, 8, (obs,), generator=g, device="cuda", dtype=torch.int32)
        _plan(case, state)
        _store(state, 1, obs, n_kv, hd, S + 8)
        state["k"].zero_()
        state["v"].zero_()
        state["q"] = torch.empty((obs, n_q, S, hd), dtype=torch.bfloat16, device="cuda")
        return state
    rows = case["rows"]
    if case["kind"] == "evict":
        L = case["layers"]
        _store(state, L, obs, n_kv, hd, rows)
        state["k"].normal_(0.0, 1.0, generator=g)
        state["v"].normal_(0.0, 1.0, generator=g)
        # weights that fall off steeply, and rows that nothing looked at
        mass = torch.exp(normal(L, obs, n_kv, rows, std=2.0))
        mass[torch.rand(mass.shape, generator=g, device="cuda") < 0.1] = 0.0
        state["mass"] = mass
        shape = (L, obs, n_kv, case["keep"])
        if own:
            import vla_cpp_b200 as vb

            state["dst"] = vb.KvStore(L, obs, n_kv, hd, case["keep"], 0)
        state["mass_out"] = torch.zeros(shape, dtype=torch.float32, device="cuda")
        state["kept"] = torch.zeros(shape, dtype=torch.int32, device="cuda")
        state["lens_out"] = torch.zeros(obs, dtype=torch.int32, device="cuda")
        return state
    S = case["tokens"]
    _store(state, 1, obs, n_kv, hd, rows)
    state["k"].normal_(0.0, 1.0, generator=g)
    state["v"].normal_(0.0, 1.0, generator=g)
    state["q"] = normal(obs, n_q, S, hd, std=1.5, dtype=torch.bfloat16)
    state["pad"] = None
    if case["pad"]:
        lens = state["lens"].tolist()
        state["pad"] = torch.tensor([_pad_of(case, n) for n in lens], dtype=torch.int32, device="cuda")
    if case["kind"] == "cross":
        state["out"] = torch.empty((obs, S, n_q * hd), dtype=torch.bfloat16, device="cuda")
        state["lse"] = torch.empty((obs, n_q, S), dtype=torch.float32, device="cuda")
    else:
        state["lse"] = _attend(state, with_out=False)[1]
        state["mass"] = torch.rand((obs, n_kv, rows), generator=g, device="cuda")
        state["mass_out"] = torch.zeros((obs, n_kv, rows), dtype=torch.float32, device="cuda")
    return state


# ------------------------------------------------------------------------------------------------- plain forms
def _visible(state, b):
    """Which rows of observation b's pages the queries may see."""
    rows = state["k"].shape[3]
    at = torch.arange(rows, device="cuda")
    seen = at < state["lens"][b]
    if state["pad"] is not None:
        seen &= (at < state["pad"][b, 0]) | (at >= state["pad"][b, 1])
    return seen


def _scores(state, b):
    """float32 [n_kv, g * S, rows] of one observation, -inf where a row is hidden."""
    n_kv, rows, hd = state["k"].shape[2:]
    q = state["q"][b].reshape(n_kv, -1, hd).float()
    s = torch.matmul(q, state["k"][0, b].float().transpose(1, 2)) * (1.0 / math.sqrt(hd))
    return s.masked_fill(~_visible(state, b), -math.inf)


def _attend(state, with_out=True):
    obs, n_q, S, hd = state["q"].shape
    n_kv = state["k"].shape[2]
    outs, lses = [], []
    for b in range(obs):
        s = _scores(state, b)
        top = s.amax(-1, keepdim=True)
        top = torch.where(top == -math.inf, torch.zeros_like(top), top)
        e = torch.exp(s - top)
        total = e.sum(-1, keepdim=True)
        lses.append((top + torch.log(total)).reshape(n_q, S))
        if with_out:
            v = state["v"][0, b].float().masked_fill(~_visible(state, b)[:, None], 0.0)
            o = torch.matmul(e, v) / torch.where(total == 0, torch.ones_like(total), total)
            outs.append(o.reshape(n_q, S, hd).transpose(0, 1).reshape(S, n_q * hd).bfloat16())
    return (torch.stack(outs) if with_out else None), torch.stack(lses)


def _plain_rope(state):
    case = state["case"]
    n_q, n_kv, hd = HEADS[case["heads"]]
    obs, S, rot = case["obs"], case["tokens"], case["rot"]
    x = state["x"].float().reshape(obs, S, n_q + 2 * n_kv, hd)

    def normed(h, w):
        return h / torch.sqrt((h * h).mean(-1, keepdim=True) + 1e-6) * w

    angle = state["pos"].double()[..., None] * state["freqs"]
    c = (torch.cos(angle) * state["mscale"]).float()[:, :, None]
    s = (torch.sin(angle) * state["mscale"]).float()[:, :, None]

    def turned(h):
        r = h[..., :rot]
        a, b = (r[..., 0::2], r[..., 1::2]) if case["interleaved"] else (r[..., :rot // 2], r[..., rot // 2:])
        a, b = a * c - b * s, b * c + a * s
        r = torch.stack((a, b), -1).flatten(-2) if case["interleaved"] else torch.cat((a, b), -1)
        return torch.cat((r, h[..., rot:]), -1)

    q = turned(normed(x[:, :, :n_q], state["q_w"]))
    k = turned(normed(x[:, :, n_q:n_q + n_kv], state["k_w"]))
    v = x[:, :, n_q + n_kv:]
    live = torch.arange(S, device="cuda")[None] < state["lens"][:, None]
    q = torch.where(live[:, :, None, None], q, torch.zeros_like(q))
    state["q"].copy_(q.transpose(1, 2))
    b, t = torch.nonzero(live, as_tuple=True)
    row = state["row0"][b].long() + t
    state["k"][0, b, :, row] = k[b, t].bfloat16()
    state["v"][0, b, :, row] = v[b, t].bfloat16()
    return state["q"], state["k"], state["v"]


def _plain_mass(state):
    out = state["mass_out"]
    obs, n_q, S, hd = state["q"].shape
    n_kv, rows = state["k"].shape[2:4]
    for b in range(obs):
        lse = state["lse"][b].reshape(n_kv, -1, 1)
        w = torch.exp(_scores(state, b) - torch.where(lse == -math.inf, torch.full_like(lse, math.inf), lse))
        new = 0.5 * state["mass"][b] + w.sum(1)
        out[b] = torch.where(torch.arange(rows, device="cuda") < state["lens"][b], new, out[b])
    return out


def _plain_evict(state):
    case = state["case"]
    L, obs, n_kv, rows, hd = state["k"].shape
    keep = case["keep"]
    n = state["lens"].long()[None, :, None, None]
    at = torch.arange(rows, device="cuda")
    rank = torch.where(torch.isnan(state["mass"]), torch.full_like(state["mass"], -math.inf), state["mass"]).double()
    rank = torch.where((at < case["sink"]) | (at >= n - case["recent"]), torch.full_like(rank, math.inf), rank)
    # hidden rows sort behind everything: a first key of whether the row exists
    by_mass = torch.sort(rank, dim=-1, descending=True, stable=True).indices
    by_life = torch.sort(torch.gather((at < n).expand(rank.shape).int(), -1, by_mass), dim=-1, descending=True, stable=True).indices
    chosen = torch.gather(by_mass, -1, by_life)[..., :keep]
    slot = torch.arange(keep, device="cuda")
    count = torch.clamp(n, max=keep)
    chosen = torch.where(slot < count, chosen, torch.full_like(chosen, rows)).sort(-1).values
    live = slot < count
    src = torch.where(live, chosen, torch.zeros_like(chosen))
    pick = src[..., None].expand(*src.shape, hd)
    k = torch.gather(state["k"], 3, pick) * live[..., None]
    v = torch.gather(state["v"], 3, pick) * live[..., None]
    mass = torch.gather(state["mass"], 3, src) * live
    kept = torch.where(live, chosen, torch.full_like(chosen, -1)).int()
    return k, v, mass, kept, torch.clamp(state["lens"], max=keep)


# ------------------------------------------------------------------------------------------------- one pass
def run(state):
    case = state["case"]
    kind = case["kind"]
    if not own:
        if kind == "rope":
            return _plain_rope(state)
        if kind == "cross":
            return _attend(state)
        return _plain_mass(state) if kind == "mass" else _plain_evict(state)
    import vla_cpp_b200 as vb

    if kind == "rope":
        n_q = HEADS[case["heads"]][0]
        vb.qk_norm_rope_append(state["store"], 0, state["x"], case["tokens"], n_q, state["freqs"], q_norm=state["q_w"],
                               k_norm=state["k_w"], eps=1e-6, interleaved=case["interleaved"], mscale=state["mscale"],
                               pos=state["pos"], row0=state["row0"], n_tok=state["lens"] if case["ragged"] else None,
                               q_out=state["q"])
        return state["q"], state["k"], state["v"]
    if kind == "cross":
        vb.cross_attention(state["store"], 0, state["q"], lens=state["lens"], pad_ranges=state["pad"], out=state["out"],
                           lse=state["lse"])
        return state["out"], state["lse"]
    if kind == "mass":
        return vb.key_mass(state["store"], 0, state["q"], state["lse"], lens=state["lens"], pad_ranges=state["pad"], decay=0.5,
                           mass=state["mass"], out=state["mass_out"])
    vb.kv_evict(state["store"], state["dst"], state["mass"], case["keep"], lens=state["lens"], sink=case["sink"],
                recent=case["recent"], mass_out=state["mass_out"], kept=state["kept"], lens_out=state["lens_out"])
    return state["dst"].k, state["dst"].v, state["mass_out"], state["kept"], state["lens_out"]


# ------------------------------------------------------------------------------------------------- costs
def work(case):
    n_q, n_kv, hd = HEADS[case["heads"]]
    obs, lens = case["obs"], _lens(case)
    if case["kind"] == "rope":
        S, live = case["tokens"], sum(lens)
        width = (n_q + 2 * n_kv) * hd
        read = live * width * (4 if case["f32"] else 2) + live * 4 + obs * 8 + 8 * hd + 4 * case["rot"]
        written = obs * S * n_q * hd * 2 + live * 2 * n_kv * hd * 2
        return {"bytes": read + written, "flops": live * (n_q + n_kv) * (4 * hd + 3 * case["rot"])}
    if case["kind"] == "evict":
        pages = case["layers"] * n_kv
        kept = sum(min(n, case["keep"]) for n in lens)
        moved = 2 * 2 * kept * hd * 2 * pages
        small = pages * (sum(lens) * 4 + obs * case["keep"] * 8) + obs * 8
        return {"bytes": moved + small, "flops": pages * sum(lens)}
    S = case["tokens"]
    seen = sum(_seen(case))
    queries = obs * n_q * S
    if case["kind"] == "cross":
        return {"bytes": queries * hd * 4 + queries * 4 + 2 * seen * n_kv * hd * 2 + obs * 4,
                "flops": 4 * n_q * S * seen * hd}
    return {"bytes": queries * hd * 2 + queries * 4 + seen * n_kv * hd * 2 + sum(lens) * n_kv * 8 + obs * 4,
            "flops": 2 * n_q * S * seen * hd}


# ------------------------------------------------------------------------------------------------- from the definitions
def exact(case, seed):
    n_q, n_kv, hd = HEADS[case["heads"]]
    obs = case["obs"]
    if case["kind"] in ("cross", "mass") and work(case)["flops"] > 6e11:
        return None
    st = prepare(case, seed)
    lens = st["lens"].tolist()
    if case["kind"] == "rope":
        return _exact_rope(case, st, lens)
    if case["kind"] == "evict":
        return _exact_evict(case, st, lens)
    g, S = n_q // n_kv, case["tokens"]
    out = torch.zeros((obs, S, n_q * hd), dtype=torch.float64, device="cuda")
    lse = torch.full((obs, n_q, S), -math.inf, dtype=torch.float64, device="cuda")
    mass = st["mass_out"].double() if case["kind"] == "mass" else None
    for b in range(obs):
        rows = list(range(lens[b]))
        if case["pad"]:
            lo, hi = _pad_of(case, lens[b])
            rows = rows[:lo] + rows[hi:]
        if mass is not None:
            mass[b, :, :lens[b]] = 0.5 * st["mass"][b, :, :lens[b]].double()
        if not rows:
            continue
        at = torch.tensor(rows, device="cuda")
        for h in range(n_q):
            k = st["k"][0, b, h // g].index_select(0, at).double()
            z = torch.einsum("sd,nd->sn", st["q"][b, h].double(), k) / hd ** 0.5
            if mass is not None:
                mass[b, h // g].index_add_(0, at, torch.exp(z - st["lse"][b, h].double()[:, None]).sum(0))
                continue
            lse[b, h] = torch.logsumexp(z, -1)
            p = torch.exp(z - lse[b, h][:, None])
            out[b, :, h * hd:(h + 1) * hd] = torch.einsum("sn,nd->sd", p, st["v"][0, b, h // g].index_select(0, at).double())
    return mass if mass is not None else (out, lse)


def _exact_rope(case, st, lens):
    n_q, n_kv, hd = HEADS[case["heads"]]
    obs, S, rot = case["obs"], case["tokens"], case["rot"]
    f, mscale = _frequencies(rot, case["scaling"], case["factor"])
    x = st["x"].double().view(obs, S, -1, hd)
    # each rotated pair as one complex number, turned by mscale * exp(i angle)
    turn = torch.polar(torch.full((obs, S, rot // 2), mscale, dtype=torch.float64, device="cuda"),
                       st["pos"].double().unsqueeze(-1) * torch.tensor(f, dtype=torch.float64, device="cuda")).unsqueeze(2)
    i = torch.arange(rot // 2, device="cuda")
    re, im = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + rot // 2)

    def head(h, w):
        y = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + 1e-6) * w.double()
        z = torch.complex(y[..., re], y[..., im]) * turn
        y[..., re], y[..., im] = z.real, z.imag
        return y

    q = head(x[:, :, :n_q], st["q_w"]).permute(0, 2, 1, 3).contiguous()
    k, v = head(x[:, :, n_q:n_q + n_kv], st["k_w"]), x[:, :, n_q + n_kv:]
    k_pages, v_pages = st["k"].double(), st["v"].double()
    for b, first in enumerate(st["row0"].tolist()):
        q[b, :, lens[b]:] = 0.0
        k_pages[0, b, :, first:first + lens[b]] = k[b, :lens[b]].transpose(0, 1)
        v_pages[0, b, :, first:first + lens[b]] = v[b, :lens[b]].transpose(0, 1)
    return q, k_pages, v_pages


def _exact_evict(case, st, lens):
    keep, L, n_kv = case["keep"], case["layers"], HEADS[case["heads"]][1]
    shape = (L, case["obs"], n_kv, keep)
    k = torch.zeros((*shape, st["k"].shape[-1]), dtype=torch.float64, device="cuda")
    v = torch.zeros_like(k)
    mass = torch.zeros(shape, dtype=torch.float64, device="cuda")
    kept = torch.full(shape, -1, dtype=torch.int32, device="cuda")
    for b, n in enumerate(lens):
        m = st["mass"][:, b, :, :n].double().reshape(L * n_kv, n).clone()
        m[:, :case["sink"]] = math.inf
        m[:, max(n - case["recent"], 0):] = math.inf
        if n == 0:
            continue
        # a row stays if fewer than `keep` rows are heavier, or as heavy and in front of it
        at = torch.arange(n, device="cuda")
        for page in range(L * n_kv):
            w = m[page]
            ahead = (w[None] > w[:, None]).sum(1) + ((w[None] == w[:, None]) & (at[None] < at[:, None])).sum(1)
            rows = torch.nonzero(ahead < keep).flatten()
            l, h, c = page // n_kv, page % n_kv, rows.numel()
            k[l, b, h, :c] = st["k"][l, b, h].index_select(0, rows).double()
            v[l, b, h, :c] = st["v"][l, b, h].index_select(0, rows).double()
            mass[l, b, h, :c] = st["mass"][l, b, h].index_select(0, rows).double()
            kept[l, b, h, :c] = rows.int()
    return k, v, mass, kept, torch.tensor([min(n, keep) for n in lens], dtype=torch.int32, device="cuda")
