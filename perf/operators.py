"""Measured cases of the cache operators: rotary positions, attention with modified scores, eviction.

`run` computes an operator either in its plain form (elementary torch operations in 32 bits, angles in
64) or, where `own` is true, through the library's entry points.  A case is a dict of plain values; its
ragged lengths follow from its own `mix`, its values from the seed.  K and V are N(0, 1) like the rows of
the other benchmarks, pools are paged in 16-token blocks in shuffled order.
"""
import importlib.util
import math
import os
import random
import sys

import torch

own = False

BT = 16  # tokens of a block
DT = {"bf16": torch.bfloat16, "f32": torch.float32}


# ---- cases ---------------------------------------------------------------------------------------------

def listed():
    return [
        # one decoder layer's projections of a decode batch: 64 sequences, one token each (latency)
        dict(name="rope_tokens_64", op="rope_rows", rows=64, heads=10, kv_heads=10, head_dim=128, dtype="f32", pool="bf16",
             layout="half", rotary=128, scaling="none", far=20000, slots=64, mix=1),
        # an admission wave of 16 pages of 1024 vision tokens, q/k/v in one projection row, half of the head rotated, long context
        dict(name="rope_write_pages", op="rope_write", rows=16384, heads=10, kv_heads=10, head_dim=128, dtype="bf16", pool="bf16",
             layout="interleaved", rotary=64, scaling="ramp", far=100000, slots=16, mix=2),
        # grouped heads, fp32 rows and pool, far positions, ragged requests
        dict(name="rope_write_ragged_f32", op="rope_write", rows=1537, heads=16, kv_heads=4, head_dim=64, dtype="f32", pool="f32",
             layout="half", rotary=48, scaling="bands", far=1000000, slots=5, mix=3),
        # one sequence, one page, a capped score (latency)
        dict(name="decode_one", op="decode", rows=1, prefix=273, window=128, heads=10, kv_heads=10, head_dim=128, pool="bf16",
             out="f32", cap=30.0, bias=False, pages=1, shared=False, mass=False, mix=4),
        # 64 sequences transcribe the pages of one shared document of 2048 tokens, each sees its own page and its window of 1024
        dict(name="decode_pages_64", op="decode", rows=64, prefix=2048, window=1024, heads=10, kv_heads=10, head_dim=128, pool="bf16",
             out="bf16", cap=0.0, bias=True, pages=8, shared=True, mass=False, mix=5),
        # few sequences, long caches, grouped heads, cap and bias together
        dict(name="decode_long_grouped", op="decode", rows=6, prefix=20000, window=4096, heads=16, kv_heads=4, head_dim=128, pool="bf16",
             out="f32", cap=50.0, bias=True, pages=1, shared=False, mass=False, mix=6),
        # the step of an evicting engine: 48 sequences of their own long prefixes, attention weights accumulated
        dict(name="decode_mass_48", op="decode", rows=48, prefix=2500, window=256, heads=10, kv_heads=10, head_dim=128, pool="bf16",
             out="bf16", cap=0.0, bias=False, pages=1, shared=False, mass=True, mix=7),
        # vision rows of 4 documents of pages that see themselves in both directions, capped scores
        dict(name="prefill_pages", op="prefill", requests=4, prefix=2184, window=1024, text=0, heads=10, kv_heads=10, head_dim=128,
             pool="bf16", rows_dtype="bf16", out="bf16", cap=50.0, bias=False, pages=8, mix=8),
        # text prompts of up to 2048 tokens over a prefix of 1056 and a window of 1024, distance bias
        dict(name="prefill_text_bias", op="prefill", requests=8, prefix=1056, window=1024, text=2048, heads=10, kv_heads=10, head_dim=128,
             pool="bf16", rows_dtype="f32", out="f32", cap=0.0, bias=True, pages=1, mix=9),
        # a short wave on fp32 KV with grouped heads of 64 (causal pages, odd lengths)
        dict(name="prefill_small_f32", op="prefill", requests=3, prefix=157, window=64, text=0, heads=4, kv_heads=2, head_dim=64,
             pool="f32", rows_dtype="f32", out="f32", cap=20.0, bias=True, pages=3, mix=10),
        # one sequence of one page gives up half of its vision tokens (latency)
        dict(name="evict_one", op="evict", slots=1, prefix=273, keep=128, sinks=4, recent=16, layers=12, heads=10, head_dim=128, pool="bf16", mix=11),
        # 8 sequences of 4096 vision tokens keep a quarter, 6 layers
        dict(name="evict_wave", op="evict", slots=8, prefix=4096, keep=1024, sinks=16, recent=64, layers=6, heads=10, head_dim=128, pool="bf16", mix=12),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rope_rows", "rope_write", "decode", "decode", "prefill", "evict"])
    mix = rng.randrange(1 << 30)
    if op in ("rope_rows", "rope_write"):
        head_dim = rng.choice([64, 128])
        heads, kv_heads = rng.choice([(10, 10), (16, 4), (4, 2)])
        return dict(op=op, rows=_spread(rng, 1, 16384), heads=heads, kv_heads=kv_heads, head_dim=head_dim, dtype=rng.choice(["bf16", "f32"]),
                    pool=rng.choice(["bf16", "f32"]), layout=rng.choice(["half", "interleaved"]),
                    rotary=rng.choice([head_dim, head_dim // 2, 3 * head_dim // 4]), scaling=rng.choice(["none", "linear", "base", "ramp", "bands"]),
                    far=_spread(rng, 1000, 1000000), slots=_spread(rng, 1, 16), mix=mix)
    if op == "decode":
        heads, kv_heads = rng.choice([(10, 10), (10, 10), (16, 4), (4, 2)])
        shared = rng.random() < 0.4
        prefix = _spread(rng, 64, 20000)
        window = _spread(rng, 16, 4096)
        rows = max(1, min(_spread(rng, 1, 96), 150000 // (prefix + window)))
        return dict(op=op, rows=rows, prefix=prefix, window=window, heads=heads, kv_heads=kv_heads, head_dim=rng.choice([64, 128, 128]),
                    pool=rng.choice(["bf16", "bf16", "f32"]), out=rng.choice(["bf16", "f32"]), cap=rng.choice([0.0, 20.0, 50.0]),
                    bias=rng.random() < 0.5, pages=rng.choice([1, 1, 4, 9]), shared=shared, mass=rng.random() < 0.4, mix=mix)
    if op == "prefill":
        text = rng.choice([0, 1]) * _spread(rng, 16, 2048)
        return dict(op=op, requests=_spread(rng, 1, 6), prefix=_spread(rng, 64, 2048), window=_spread(rng, 16, 1024), text=text, heads=10, kv_heads=10,
                    head_dim=128, pool="bf16", rows_dtype=rng.choice(["bf16", "f32"]), out=rng.choice(["bf16", "f32"]),
                    cap=rng.choice([0.0, 30.0]), bias=rng.random() < 0.5, pages=rng.choice([1, 2, 7]), mix=mix)
    prefix = _spread(rng, 64, 4096)
    return dict(op=op, slots=_spread(rng, 1, 8), prefix=prefix, keep=max(1, int(prefix * rng.uniform(0.1, 0.9))), sinks=rng.choice([0, 4, 16]),
                recent=rng.choice([0, 16, 64]), layers=_spread(rng, 1, 6), heads=10, head_dim=rng.choice([64, 128]),
                pool=rng.choice(["bf16", "f32"]), mix=mix)


# ---- ragged lengths: from the case alone ---------------------------------------------------------------

def _page_edges(n, pages):
    """Cuts [0, n) into `pages` pages of nearly equal, odd sizes."""
    return [round(i * n / pages) for i in range(pages + 1)]


def _shape(c):
    rng = random.Random(c["mix"])
    if c["op"] in ("rope_rows", "rope_write"):
        cuts = sorted(rng.randrange(c["rows"] + 1) for _ in range(c["slots"] - 1))
        return [b - a for a, b in zip([0] + cuts, cuts + [c["rows"]])]  # rows of every slot
    if c["op"] == "decode":
        rows = []
        for r in range(c["rows"]):
            p = c["prefix"] if c["shared"] else max(1, c["prefix"] - rng.randrange(c["prefix"] // 8 + 1))
            text = c["window"] if rng.random() < 0.75 else rng.randrange(1, c["window"] + 1)  # most windows have wrapped
            ring = rng.randrange(c["window"]) if text == c["window"] else 0
            page = rng.randrange(c["pages"])
            e = _page_edges(p, c["pages"])
            past = rng.randrange(c["window"] + 1) if text == c["window"] else 0  # text tokens the window has dropped
            rows.append((p, text, ring, e[page], e[page + 1], p + text + past - 1))
        return rows
    if c["op"] == "prefill":
        out = []
        for r in range(c["requests"]):
            p = max(1, c["prefix"] - rng.randrange(c["prefix"] // 4 + 1))
            t = rng.randrange(max(1, c["text"] // 4), c["text"] + 1) if c["text"] else 0
            out.append((p, t))
        return out
    return [max(1, c["prefix"] - rng.randrange(c["prefix"] // 8 + 1)) for _ in range(c["slots"])]


def _bytes(name):
    return 2 if name == "bf16" else 4


def work(case):
    c, s = case, _shape(case)
    if c["op"] in ("rope_rows", "rope_write"):
        kv = c["kv_heads"] * c["head_dim"]
        q = c["heads"] * c["head_dim"]
        if c["op"] == "rope_rows":
            b = c["rows"] * (2 * (q + kv) * _bytes(c["dtype"]) + 4)
        else:
            b = c["rows"] * ((2 * q + 2 * kv) * _bytes(c["dtype"]) + 2 * kv * _bytes(c["pool"]) + 12)
        return {"bytes": b, "flops": c["rows"] * (c["heads"] + c["kv_heads"]) * c["rotary"] * 3}
    if c["op"] == "decode":
        tok = 2 * c["kv_heads"] * c["head_dim"] * _bytes(c["pool"])
        pairs = sum(hi - lo + text for _, text, _, lo, hi, _ in s)
        if c["shared"]:
            seen = set()
            for _, _, _, lo, hi, _ in s:
                seen.add((lo, hi))
            toks = sum(hi - lo for lo, hi in seen) + sum(r[1] for r in s)
        else:
            toks = pairs
        b = toks * tok + c["rows"] * c["heads"] * c["head_dim"] * (4 + _bytes(c["out"]))
        if c["mass"]:
            b += sum(r[0] for r in s) * 8
        return {"bytes": b, "flops": pairs * c["heads"] * c["head_dim"] * 4}
    if c["op"] == "prefill":
        kv = 2 * c["kv_heads"] * c["head_dim"] * _bytes(c["pool"])
        pairs = rows = toks = 0
        for p, t in s:
            if c["text"]:
                pairs += t * p + sum(min(i + 1, c["window"]) for i in range(t))
                rows += t
                toks += p + t
            else:
                e = _page_edges(p, c["pages"])
                pairs += sum((b - a) ** 2 for a, b in zip(e, e[1:]))
                rows += p
                toks += p
        b = toks * kv + rows * c["heads"] * c["head_dim"] * (_bytes(c["rows_dtype"]) + _bytes(c["out"]))
        return {"bytes": b, "flops": pairs * c["heads"] * c["head_dim"] * 4}
    kept = sum(min(p, c["keep"]) for p in s)
    return {"bytes": sum(s) * 4 + kept * (4 + c["layers"] * 2 * 2 * c["heads"] * c["head_dim"] * _bytes(c["pool"])), "flops": sum(s)}


# ---- inputs --------------------------------------------------------------------------------------------

ROPE = dict(theta=10000.0, factor=8.0, orig=4096.0)
BANDS = dict(none=(0.0, 0.0), linear=(0.0, 0.0), base=(0.0, 0.0), ramp=(1.0, 32.0), bands=(1.0, 4.0))  # (low, high)


def _amplitude(c):
    return 0.1 * math.log(ROPE["factor"]) + 1.0 if c["scaling"] == "ramp" else 1.0


def _slopes(heads):
    """Geometric slopes 2^(-8 (h + 1) / heads)."""
    return [2.0 ** (-8.0 * (h + 1) / heads) for h in range(heads)]


def _tables(lens, ring_blocks, shared, gen):
    """Block table [slots, stride] in shuffled block order: prefix blocks, then ring blocks; and the block count."""
    nb = [(p + BT - 1) // BT for p in lens]
    pre = max(nb) if shared else sum(nb)
    total = pre + ring_blocks * len(lens)
    ids = torch.randperm(total, generator=gen, device="cuda").to(torch.int32)
    table = torch.full((len(lens), max(nb) + ring_blocks), -1, dtype=torch.int32, device="cuda")
    at = pre
    p0 = 0
    for i, n in enumerate(nb):
        table[i, :n] = ids[:n] if shared else ids[p0:p0 + n]
        p0 += 0 if shared else n
        table[i, n:n + ring_blocks] = ids[at:at + ring_blocks]
        at += ring_blocks
    return table, total


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _inputs(c, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed * 7919 + 13)
    normal = lambda *shape, dtype=torch.float32: torch.randn(*shape, generator=gen, device="cuda", dtype=dtype)
    s = _shape(c)
    st = dict(case=c, shape=s)
    if c["op"] in ("rope_rows", "rope_write"):
        q, kv = c["heads"] * c["head_dim"], c["kv_heads"] * c["head_dim"]
        dt = DT[c["dtype"]]
        qkv = normal(c["rows"], q + 2 * kv, dtype=dt)  # one projection row: q, k, v
        st.update(q=qkv[:, :q], k=qkv[:, q:q + kv], v=qkv[:, q + kv:], q_out=torch.empty(c["rows"], q, dtype=dt, device="cuda"))
        first = torch.randint(0, max(1, c["far"] - c["rows"]), (c["slots"],), generator=gen, device="cuda")
        slot = torch.repeat_interleave(torch.arange(c["slots"], device="cuda"), torch.tensor(s, device="cuda"))
        pos = torch.cat([torch.arange(n, device="cuda") for n in s])
        st.update(d_slots=slot.to(torch.int32), d_pos=pos.to(torch.int32), d_positions=(pos + first[slot]).to(torch.int32))
        if c["op"] == "rope_rows":
            st.update(k_out=torch.empty(c["rows"], kv, dtype=dt, device="cuda"))
        else:
            table, total = _tables(s, 0, False, gen)
            shape = (total, c["kv_heads"], BT, c["head_dim"])
            st.update(table=table, k_pool=torch.zeros(shape, dtype=DT[c["pool"]], device="cuda"),
                      v_pool=torch.zeros(shape, dtype=DT[c["pool"]], device="cuda"), d_prefill=_ints(s))
        return st
    if c["op"] == "decode":
        ring_blocks = (c["window"] + BT - 1) // BT
        table, total = _tables([r[0] for r in s], ring_blocks, c["shared"], gen)
        shape = (total, c["kv_heads"], BT, c["head_dim"])
        order = list(range(c["rows"]))
        random.Random(c["mix"] + 1).shuffle(order)  # batch row r serves slot order[r]
        stride = table.shape[1] * BT
        st.update(table=table, k_pool=normal(*shape, dtype=DT[c["pool"]]), v_pool=normal(*shape, dtype=DT[c["pool"]]),
                  q=normal(c["rows"], c["heads"] * c["head_dim"]), order=order, d_slots=_ints(order),
                  d_prefill=_ints([r[0] for r in s]), d_len=_ints([r[0] + r[1] for r in s]), d_ring=_ints([r[2] for r in s]),
                  d_lo=_ints([s[o][3] for o in order]), d_hi=_ints([s[o][4] for o in order]), d_q_pos=_ints([s[o][5] for o in order]),
                  slopes=torch.tensor(_slopes(c["heads"]), device="cuda"),
                  out=torch.empty(c["rows"], c["heads"] * c["head_dim"], dtype=DT[c["out"]], device="cuda"))
        if c["mass"]:
            st.update(mass_in=torch.rand(c["rows"], stride, generator=gen, device="cuda") * 3, mass_out=torch.zeros(c["rows"], stride, device="cuda"))
        return st
    if c["op"] == "prefill":
        table, total = _tables([p for p, _ in s], 0, False, gen)
        shape = (total, c["kv_heads"], BT, c["head_dim"])
        rows = sum(t if c["text"] else p for p, t in s)
        st.update(table=table, k_pool=normal(*shape, dtype=DT[c["pool"]]), v_pool=normal(*shape, dtype=DT[c["pool"]]),
                  q=normal(rows, c["heads"] * c["head_dim"], dtype=DT[c["rows_dtype"]]), d_prefill=_ints([p for p, _ in s]),
                  slopes=torch.tensor(_slopes(c["heads"]), device="cuda"), rows=rows,
                  out=torch.empty(rows, c["heads"] * c["head_dim"], dtype=DT[c["out"]], device="cuda"))
        slots, pos, lo, hi, block0, requests = [], [], [], [], [], []
        at = tb = 0
        for i, (p, t) in enumerate(s):
            if c["text"]:
                slots += [i] * t
                pos += range(t)
                lo += [0] * t
                hi += [p] * t
                block0 += [tb] * t
                requests.append((at, t, i, 1, 0, tb))
                tb += (t + BT - 1) // BT
                at += t
            else:
                e = _page_edges(p, c["pages"])
                slots += [i] * p
                pos += range(p)
                for a, b in zip(e, e[1:]):
                    lo += [a] * (b - a)
                    hi += [b] * (b - a)
                block0 += [0] * p
                requests.append((at, p, i, 0, 0, 0))
                at += p
        st.update(d_slots=_ints(slots), d_pos=_ints(pos), d_lo=_ints(lo), d_hi=_ints(hi), d_block0=_ints(block0), requests=requests,
                  d_q_pos=_ints([x + (s[i][0] if c["text"] else 0) for x, i in zip(pos, slots)]), text_blocks=tb)
        if c["text"]:
            shape = (tb, c["kv_heads"], BT, c["head_dim"])
            st.update(k_text=normal(*shape, dtype=DT[c["pool"]]), v_text=normal(*shape, dtype=DT[c["pool"]]))
        return st
    table, total = _tables(s, 0, False, gen)
    new = (min(c["keep"], max(s)) + BT - 1) // BT
    shape = (total + new * c["slots"], c["heads"], BT, c["head_dim"])
    mass = -torch.log(torch.rand(c["slots"], table.shape[1] * BT, generator=gen, device="cuda").clamp_min(1e-7))
    mass = torch.where(mass < 0.3, torch.zeros_like(mass), mass)  # tokens that no row has looked at
    mass = torch.where(mass > 1.5, mass, (mass * 64).round() / 64)  # and ties
    st.update(table=table, mass=mass, d_prefill=_ints(s), d_slots=_ints(list(range(c["slots"]))),
              k_pools=[normal(*shape, dtype=DT[c["pool"]]) for _ in range(c["layers"])],
              v_pools=[normal(*shape, dtype=DT[c["pool"]]) for _ in range(c["layers"])],
              d_new=(total + torch.randperm(new * c["slots"], generator=gen, device="cuda").to(torch.int32)).reshape(c["slots"], new).contiguous(),
              d_keep=torch.empty(c["slots"], c["keep"], dtype=torch.int32, device="cuda"), d_keep_len=torch.empty(c["slots"], dtype=torch.int32, device="cuda"))
    return st


def _package():
    if "uocr_b200" not in sys.modules:
        root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
        spec = importlib.util.spec_from_file_location("uocr_b200", os.path.join(root, "unlimited-ocr.cpp_b200", "__init__.py"))
        mod = importlib.util.module_from_spec(spec)
        sys.modules["uocr_b200"] = mod
        spec.loader.exec_module(mod)
    return sys.modules["uocr_b200"]


def prepare(case, seed):
    c, st = case, _inputs(case, seed)
    if not own:
        return st
    b = st["b"] = _package()
    layer = lambda k, v: b.PagedLayer(k.shape[0], k.shape[1], k.shape[3], b.BF16 if k.dtype == torch.bfloat16 else b.F32, st["table"], pools=(k, v))
    if c["op"] in ("rope_rows", "rope_write"):
        low, high = BANDS[c["scaling"]]
        st["rope"] = b.Rope(layout=c["layout"], rotary_dim=c["rotary"], theta=ROPE["theta"], scaling=c["scaling"], factor=ROPE["factor"],
                            orig_context=ROPE["orig"], low=low, high=high, amplitude=_amplitude(c))
        st["ws"] = b.Workspace(c["rows"])
        if c["op"] == "rope_write":
            st["layer"] = layer(st["k_pool"], st["v_pool"])
    elif c["op"] == "decode":
        st["layer"] = layer(st["k_pool"], st["v_pool"])
        st["ws"] = b.Workspace(c["rows"])
        st["ws"].set_out_dtype(b.BF16 if c["out"] == "bf16" else b.F32)
        paged = c["pages"] > 1
        st["score"] = b.Score(softcap=c["cap"], slopes=st["slopes"] if c["bias"] else None, d_q_pos=st["d_q_pos"] if c["bias"] else None,
                              d_lo=st["d_lo"] if paged else None, d_hi=st["d_hi"] if paged else None)
        st["mass"] = b.Mass(st["mass_in"], st["mass_out"], c["rows"], c["heads"], decay=0.5) if c["mass"] else None
    elif c["op"] == "prefill":
        st["layer"] = layer(st["k_pool"], st["v_pool"])
        st["ws"] = b.Workspace(st["rows"])
        st["ws"].set_out_dtype(b.BF16 if c["out"] == "bf16" else b.F32)
        vision = not c["text"]
        st["score"] = b.Score(softcap=c["cap"], slopes=st["slopes"] if c["bias"] else None, d_q_pos=st["d_q_pos"] if c["bias"] else None,
                              d_lo=st["d_lo"] if vision else None, d_hi=st["d_hi"] if vision else None)
        st["tc"] = c["pool"] == "bf16" and c["head_dim"] == 128
        if st["tc"]:  # the tile plan is shared by the layers of a pass
            st["tiles"] = b.make_prefill_tiles(st["requests"])
            b.prefill_plan_scored_tc(st["score"], st["tiles"], st["d_prefill"], c["window"], st["ws"])
    else:
        st["ws"] = b.Workspace(c["slots"])
        st["layers"] = b.layer_array([layer(k, v) for k, v in zip(st["k_pools"], st["v_pools"])])
    return st


# ---- one pass ------------------------------------------------------------------------------------------

def run(st):
    c = st["case"]
    return (_own if own else _plain)[c["op"]](st, c)


def _own_rope_rows(st, c):
    st["b"].rope_rows(st["rope"], st["q"], st["k"], st["q_out"], st["k_out"], st["d_positions"], c["heads"], c["kv_heads"], c["head_dim"])
    return st["q_out"], st["k_out"]


def _own_rope_write(st, c):
    st["b"].rope_write_prefill_paged(st["layer"], st["rope"], st["q"], st["k"], st["v"], st["q_out"], st["d_positions"], st["d_slots"], st["d_pos"],
                                     c["heads"], st["ws"])
    return st["q_out"], st["k_pool"], st["v_pool"]


def _own_decode(st, c):
    st["b"].attention_scored_batch_paged(st["layer"], st["score"], st["q"], st["d_len"], st["d_ring"], st["d_prefill"], st["d_slots"], c["rows"],
                                         c["window"], c["heads"], st["out"], st["ws"], mass=st["mass"])
    return (st["out"], st["mass_out"]) if c["mass"] else st["out"]


def _own_prefill(st, c):
    b = st["b"]
    kt, vt = (st["k_text"], st["v_text"]) if c["text"] else (None, None)
    if st["tc"]:
        b.prefill_attention_scored_tc(st["layer"], kt, vt, st["text_blocks"], st["score"], st["q"], st["d_prefill"], st["tiles"], c["window"],
                                      c["heads"], st["out"], st["ws"], reuse_plan=True)
    elif c["text"]:
        b.prefill_text_scored_paged(st["layer"], kt, vt, st["text_blocks"], st["score"], st["q"], st["d_prefill"], st["d_slots"], st["d_pos"],
                                    st["d_block0"], st["rows"], c["window"], c["heads"], st["out"], st["ws"])
    else:
        b.attention_scored_ragged_paged(st["layer"], st["score"], st["q"], st["d_prefill"], st["d_slots"], st["d_pos"], st["rows"], c["heads"],
                                        st["out"], st["ws"])
    return st["out"]


def _own_evict(st, c):
    b = st["b"]
    b.evict_select(st["mass"], st["d_prefill"], st["d_slots"], c["slots"], c["keep"], c["sinks"], c["recent"], st["d_keep"], st["d_keep_len"])
    b.evict_compact_paged_layers(st["layers"], st["d_prefill"], st["d_slots"], c["slots"], st["d_keep"], st["d_keep_len"], st["d_new"], st["ws"])
    return st["d_keep"], st["d_keep_len"], st["k_pools"], st["v_pools"]


_own = dict(rope_rows=_own_rope_rows, rope_write=_own_rope_write, decode=_own_decode, prefill=_own_prefill, evict=_own_evict)


# ---- plain forms ---------------------------------------------------------------------------------------

def _frequencies(c):
    """Angle per position of the rotary pairs, in 64 bits."""
    r, theta, factor, orig = c["rotary"], ROPE["theta"], ROPE["factor"], ROPE["orig"]
    low, high = BANDS[c["scaling"]]
    i = torch.arange(0, r // 2, dtype=torch.float64, device="cuda")
    if c["scaling"] == "base" and r > 2:
        theta = theta * factor ** (r / (r - 2))
    f = theta ** (-2 * i / r)
    if c["scaling"] == "linear":
        return f / factor
    if c["scaling"] == "ramp":
        dim = lambda turns: r * math.log(orig / (turns * 2 * math.pi)) / (2 * math.log(theta))
        a, b = max(math.floor(dim(high)), 0), min(math.ceil(dim(low)), r - 1)
        ramp = ((i - a) / (b - a if b != a else 0.001)).clamp(0, 1)
        return f / factor * ramp + f * (1 - ramp)
    if c["scaling"] == "bands":
        turns = orig * f / (2 * math.pi)
        smooth = ((turns - low) / (high - low)).clamp(0, 1)
        return f / factor * (1 - smooth) + f * smooth
    return f


def _rotate(x, positions, c):
    """x [rows, heads, head_dim] in fp32."""
    angle = positions.double()[:, None] * _frequencies(c)
    cos, sin = (angle.cos() * _amplitude(c)).float()[:, None], (angle.sin() * _amplitude(c)).float()[:, None]
    r = c["rotary"]
    rot, rest = x[..., :r], x[..., r:]
    if c["layout"] == "half":
        a, b = rot[..., :r // 2], rot[..., r // 2:]
        rot = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    else:
        a, b = rot[..., 0::2], rot[..., 1::2]
        rot = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    return torch.cat([rot, rest], -1)


def _plain_rope_rows(st, c):
    hd = c["head_dim"]
    for x, out in ((st["q"], st["q_out"]), (st["k"], st["k_out"])):
        out.copy_(_rotate(x.float().unflatten(1, (-1, hd)), st["d_positions"], c).flatten(1))
    return st["q_out"], st["k_out"]


def _plain_rope_write(st, c):
    hd = c["head_dim"]
    st["q_out"].copy_(_rotate(st["q"].float().unflatten(1, (-1, hd)), st["d_positions"], c).flatten(1))
    k = _rotate(st["k"].float().unflatten(1, (-1, hd)), st["d_positions"], c)
    v = st["v"].float().unflatten(1, (-1, hd))
    blk, off = st["table"][st["d_slots"].long(), (st["d_pos"] // BT).long()].long(), (st["d_pos"] % BT).long()
    st["k_pool"][blk, :, off] = k.to(st["k_pool"].dtype)
    st["v_pool"][blk, :, off] = v.to(st["v_pool"].dtype)
    return st["q_out"], st["k_pool"], st["v_pool"]


def _scores(q, k, c, dist, slopes):
    """q [heads, n, d], k [kv_heads, m, d] (fp32), dist [n, m] -> modified scores [heads, n, m]."""
    g = q.shape[0] // k.shape[0]
    x = torch.matmul(q.unflatten(0, (-1, g)), k[:, None].transpose(-1, -2)).flatten(0, 1) / math.sqrt(c["head_dim"])
    if c["cap"]:
        x = c["cap"] * torch.tanh(x / c["cap"])
    if c["bias"]:
        x = x - slopes[:, None, None] * dist.abs()
    return x


def _weights(x, visible):
    x = x.masked_fill(~visible, float("-inf"))
    m = x.amax(-1, keepdim=True)
    e = torch.exp(x - torch.where(torch.isinf(m), torch.zeros_like(m), m))
    return e / e.sum(-1, keepdim=True).clamp_min(1e-30)


def _plain_decode(st, c):
    H, KH, D, W, B = c["heads"], c["kv_heads"], c["head_dim"], c["window"], c["rows"]
    cap = c["prefix"] + W
    step = max(1, (1 << 29) // (cap * KH * D * 4))  # rows per chunk: the gathered K and V of a chunk stay below 1 GB
    s = torch.arange(cap, device="cuda")
    if c["mass"]:
        st["mass_out"].zero_()
    for r0 in range(0, B, step):
        rows = slice(r0, min(B, r0 + step))
        slot = st["d_slots"][rows].long()
        P, ln, ring = st["d_prefill"][slot].long()[:, None], st["d_len"][slot].long()[:, None], st["d_ring"][slot].long()[:, None]
        in_ring = s >= P
        r = s - P
        entry = torch.where(in_ring, (P + BT - 1) // BT + r // BT, s // BT).clamp(0, st["table"].shape[1] - 1)
        blk = st["table"][slot[:, None], entry].long().clamp_min(0)
        off = torch.where(in_ring, r % BT, s % BT)
        k, v = st["k_pool"][blk, :, off].float(), st["v_pool"][blk, :, off].float()  # [rows, cap, kv_heads, d]
        visible = s < ln
        if c["pages"] > 1:
            visible = visible & (in_ring | ((s >= st["d_lo"][rows].long()[:, None]) & (s < st["d_hi"][rows].long()[:, None])))
        full = ln - P >= W
        age = torch.where(full, (ring - 1 - r) % W, ln - P - 1 - r)
        dist = torch.where(in_ring, age, st["d_q_pos"][rows].long()[:, None] - s).float()
        q = st["q"][rows].unflatten(1, (KH, H // KH, D))
        x = torch.matmul(q, k.permute(0, 2, 3, 1)).flatten(1, 2) / math.sqrt(D)  # [rows, heads, cap]
        if c["cap"]:
            x = c["cap"] * torch.tanh(x / c["cap"])
        if c["bias"]:
            x = x - st["slopes"][:, None] * dist.abs()[:, None]
        w = _weights(x, visible[:, None])
        st["out"][rows] = torch.matmul(w.unflatten(1, (KH, -1)), v.transpose(1, 2)).flatten(1).to(st["out"].dtype)
        if c["mass"]:
            n = min(cap, st["mass_out"].shape[1])
            got = 0.5 * st["mass_in"][slot, :n] + w.sum(1)[:, :n]
            st["mass_out"][slot, :n] = torch.where(in_ring[:, :n], torch.zeros_like(got), got)
    return (st["out"], st["mass_out"]) if c["mass"] else st["out"]


def _tokens(pool, blocks, n):
    """The first n tokens of a list of blocks, [kv_heads, n, d]."""
    return pool[blocks.long()].transpose(0, 1).flatten(1, 2)[:, :n]


def _plain_prefill(st, c):
    H, D = c["heads"], c["head_dim"]
    for i, (row0, n, slot, kind, _, block0) in enumerate(st["requests"]):
        p, t = st["shape"][slot]
        rows = slice(row0, row0 + n)
        nb = (p + BT - 1) // BT
        k, v = (_tokens(x, st["table"][slot, :nb], p).float() for x in (st["k_pool"], st["v_pool"]))
        pos = st["d_pos"][rows].long()[:, None]
        s = torch.arange(p, device="cuda")
        visible = (s >= st["d_lo"][rows].long()[:, None]) & (s < st["d_hi"][rows].long()[:, None])
        dist = st["d_q_pos"][rows].long()[:, None] - s
        if kind == 1:
            ids = torch.arange(block0, block0 + (t + BT - 1) // BT, device="cuda")
            k = torch.cat([k, _tokens(st["k_text"], ids, t).float()], 1)
            v = torch.cat([v, _tokens(st["v_text"], ids, t).float()], 1)
            j = torch.arange(t, device="cuda")
            visible = torch.cat([visible, (j <= pos) & (j > pos - c["window"])], 1)
            dist = torch.cat([dist, pos - j], 1)
        q = st["q"][rows].float().unflatten(1, (H, D)).transpose(0, 1)
        w = _weights(_scores(q, k, c, dist.float(), st["slopes"]), visible)
        o = torch.matmul(w.unflatten(0, (k.shape[0], -1)), v[:, None]).flatten(0, 1)
        st["out"][rows] = o.transpose(0, 1).flatten(1).to(st["out"].dtype)
    return st["out"]


def _plain_evict(st, c):
    n, keep = c["slots"], c["keep"]
    P = st["d_prefill"].long()[:, None]
    s = torch.arange(st["mass"].shape[1], device="cuda")
    key = torch.where((s < c["sinks"]) | (s >= P - c["recent"]), torch.full_like(st["mass"], float("inf")), st["mass"])
    key = key.masked_fill(s >= P, float("-inf"))
    order = torch.sort(key, dim=1, descending=True, stable=True).indices[:, :keep]
    count = P.clamp_max(keep)
    order = torch.where(torch.arange(order.shape[1], device="cuda") < count, order, torch.full_like(order, 1 << 30))
    kept = torch.full((n, keep), 1 << 30, dtype=torch.int64, device="cuda")
    kept[:, :order.shape[1]] = torch.sort(order, dim=1).values
    live = kept < (1 << 30)
    st["d_keep"].copy_(torch.where(live, kept, torch.full_like(kept, -1)))
    st["d_keep_len"].copy_(count[:, 0])
    row, j = torch.nonzero(live, as_tuple=True)
    src = kept[row, j]
    sb, so = st["table"][row, src // BT].long(), src % BT
    db, do = st["d_new"][row, j // BT].long(), j % BT
    for pool in st["k_pools"] + st["v_pools"]:
        pool[db, :, do] = pool[sb, :, so]
    return st["d_keep"], st["d_keep_len"], st["k_pools"], st["v_pools"]


_plain = dict(rope_rows=_plain_rope_rows, rope_write=_plain_rope_write, decode=_plain_decode, prefill=_plain_prefill, evict=_plain_evict)


# ---- the definition in 64 bits -------------------------------------------------------------------------

def _definition_angles(c):
    """Pair by pair, as plain numbers."""
    r, out = c["rotary"], []
    low, high = BANDS[c["scaling"]]
    s, L = ROPE["factor"], ROPE["orig"]
    for i in range(r // 2):
        base = ROPE["theta"]
        if c["scaling"] == "base" and r > 2:
            base *= s ** (r / (r - 2.0))
        f = base ** (-2.0 * i / r)
        if c["scaling"] == "linear":
            f /= s
        elif c["scaling"] == "ramp":
            edge = [r * math.log(L / (2 * math.pi * turns)) / (2 * math.log(base)) for turns in (high, low)]
            first, last = max(0, math.floor(edge[0])), min(r - 1, math.ceil(edge[1]))
            mix = min(1.0, max(0.0, (i - first) / ((last - first) or 0.001)))
            f = f * (1 - mix) + f / s * mix
        elif c["scaling"] == "bands":
            wave = 2 * math.pi / f
            if wave > L / low:
                f /= s
            elif wave >= L / high:
                mix = (L / wave - low) / (high - low)
                f = (1 - mix) * f / s + mix * f
        out.append(f)
    return torch.tensor(out, dtype=torch.float64, device="cuda")


def _definition_rotate(x, positions, c):
    """Each pair as a complex number times amplitude * e^(i angle)."""
    r, y = c["rotary"], x.double().clone()
    turn = torch.polar(torch.full((len(x), r // 2), _amplitude(c), dtype=torch.float64, device="cuda"),
                       torch.outer(positions.double(), _definition_angles(c)))
    i = torch.arange(r // 2, device="cuda")
    a, b = (i, i + r // 2) if c["layout"] == "half" else (2 * i, 2 * i + 1)
    z = torch.complex(y[:, :, a], y[:, :, b]) * turn[:, None]
    y[:, :, a], y[:, :, b] = z.real, z.imag
    return y


def _definition_softmax(x, v):
    """One row's scores x [m] over its visible tokens and their values v [m, d]."""
    e = torch.exp(x - x.max())
    return e / e.sum(), (e / e.sum()) @ v


def exact(case, seed):
    c, st = case, _inputs(case, seed)
    D = c["head_dim"]
    if c["op"] in ("rope_rows", "rope_write"):
        turn = lambda x: _definition_rotate(x.reshape(c["rows"], -1, D), st["d_positions"], c)
        if c["op"] == "rope_rows":
            return turn(st["q"]).reshape(c["rows"], -1), turn(st["k"]).reshape(c["rows"], -1)
        pools = [st["k_pool"].double(), st["v_pool"].double()]
        for slot, n in enumerate(st["shape"]):
            mine = (st["d_slots"] == slot).nonzero()[:, 0]
            for pool, x in zip(pools, (turn(st["k"]), st["v"].double().reshape(c["rows"], -1, D))):
                nb = (n + BT - 1) // BT
                flat = pool[st["table"][slot, :nb].long()].transpose(1, 2).flatten(0, 1)  # [tokens, kv_heads, d]
                flat[:n] = x[mine]
                pool[st["table"][slot, :nb].long()] = flat.unflatten(0, (nb, BT)).transpose(1, 2)
        return turn(st["q"]).reshape(c["rows"], -1), pools[0], pools[1]
    if c["op"] == "decode":
        H, group, W = c["heads"], c["heads"] // c["kv_heads"], c["window"]
        out = torch.zeros(c["rows"], H, D, dtype=torch.float64, device="cuda")
        mass = torch.zeros_like(st["mass_out"], dtype=torch.float64) if c["mass"] else None
        for r, slot in enumerate(st["order"]):
            p, text, ring, lo, hi, here = st["shape"][slot]
            if c["pages"] == 1:
                lo, hi = 0, p
            nb, rb = (p + BT - 1) // BT, (W + BT - 1) // BT
            k, v = ([pool[st["table"][slot, a:b].long()].double().transpose(1, 2).flatten(0, 1) for a, b in ((0, nb), (nb, nb + rb))]
                    for pool in (st["k_pool"], st["v_pool"]))
            k, v = torch.cat([k[0][lo:hi], k[1][:text]]), torch.cat([v[0][lo:hi], v[1][:text]])
            newest = (ring - 1) % W if text == W else text - 1
            away = [here - t for t in range(lo, hi)] + [(newest - t) % W for t in range(text)]
            away = torch.tensor(away, dtype=torch.float64, device="cuda").abs()
            for h in range(H):
                x = k[:, h // group] @ st["q"][r].double()[h * D:(h + 1) * D] / math.sqrt(D)
                if c["cap"]:
                    x = c["cap"] * torch.tanh(x / c["cap"])
                if c["bias"]:
                    x = x - _slopes(H)[h] * away
                w, out[r, h] = _definition_softmax(x, v[:, h // group])
                if c["mass"]:
                    mass[slot, lo:hi] += w[:hi - lo]
            if c["mass"]:
                mass[slot, :p] += 0.5 * st["mass_in"][slot, :p].double()
        out = out.flatten(1)
        return (out, mass) if c["mass"] else out
    if c["op"] == "prefill":
        H, group = c["heads"], c["heads"] // c["kv_heads"]
        out = torch.zeros(st["rows"], H, D, dtype=torch.float64, device="cuda")
        for row0, n, slot, kind, _, block0 in st["requests"]:
            p, t = st["shape"][slot]
            take = lambda pool, first, m: first(pool).double().transpose(1, 2).flatten(0, 1)[:m]
            fixed = lambda pool: pool[st["table"][slot, :(p + BT - 1) // BT].long()]
            k, v = take(st["k_pool"], fixed, p), take(st["v_pool"], fixed, p)
            if kind == 1:
                text = lambda pool: pool[block0:block0 + (t + BT - 1) // BT]
                k, v = torch.cat([k, take(st["k_text"], text, t)]), torch.cat([v, take(st["v_text"], text, t)])
            i, j = torch.arange(n, device="cuda")[:, None], torch.arange(p + t, device="cuda")[None]
            if kind == 1:
                hidden = (j >= p) & ((j - p > i) | (j - p <= i - c["window"]))
                away = (i + p - j).abs()  # text token j - p stands at position j
            else:
                page = torch.zeros(p, dtype=torch.int64, device="cuda")
                for e in _page_edges(p, c["pages"])[1:-1]:
                    page[e:] += 1
                hidden = page[:, None] != page[None]
                away = (i - j).abs()
            for h in range(H):
                x = st["q"][row0:row0 + n].double()[:, h * D:(h + 1) * D] @ k[:, h // group].T / math.sqrt(D)
                if c["cap"]:
                    x = c["cap"] * torch.tanh(x / c["cap"])
                if c["bias"]:
                    x = x - _slopes(H)[h] * away
                x[hidden.expand_as(x)] = -math.inf
                x = torch.exp(x - x.max(1, keepdim=True).values)
                out[row0:row0 + n, h] = (x @ v[:, h // group]) / x.sum(1, keepdim=True)
        return out.flatten(1)
    keep = torch.full((c["slots"], c["keep"]), -1, dtype=torch.int32)
    count = []
    k, v = [x.double() for x in st["k_pools"]], [x.double() for x in st["v_pools"]]
    mass = st["mass"].cpu().tolist()
    for slot, p in enumerate(st["shape"]):
        key = [math.inf if i < c["sinks"] or i >= p - c["recent"] else mass[slot][i] for i in range(p)]
        best = sorted(sorted(range(p), key=lambda i: (-key[i], i))[:c["keep"]])
        keep[slot, :len(best)] = torch.tensor(best, dtype=torch.int32)
        count.append(len(best))
        src = torch.tensor(best, device="cuda")
        nb = (p + BT - 1) // BT
        for pool in k + v:
            rows = pool[st["table"][slot, :nb].long()].transpose(1, 2).flatten(0, 1)[src]  # [kept, heads, d]
            mb = (len(best) + BT - 1) // BT
            dst = st["d_new"][slot, :mb].long()
            flat = pool[dst].transpose(1, 2).flatten(0, 1)
            flat[:len(best)] = rows
            pool[dst] = flat.unflatten(0, (mb, BT)).transpose(1, 2)
    return keep.cuda(), _ints(count), k, v
