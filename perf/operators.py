"""Performance cases of the serving operators: a quantised paged KV cache, attention over it with
a shared prefix, softmax of the head's logits, and verification of drafted tokens.

Each case is one pass as a program that serves the model makes it.  With `own` false the pass
is elementary torch operations in 32 bits (64 where a value next to a border decides); with
`own` true it is the calls of final_amd.lfm.  Activations are fp32, the framework's only type;
the cache is f32, bf16, int8 or fp8 (e4m3).  Buffers are torch tensors, passed by address.
"""
import math

import torch

own = False

HD = 64          # head dimension
VOCAB = 65536
E4M3_MAX = 448.0
FORMATS = ("f32", "bf16", "int8", "fp8")


def listed():
    return [
        # One sequence's next token into an int8 cache, and its few rows read back: latency.
        {"name": "kv_b1_int8", "kind": "kv", "fmt": "int8", "batch": 1, "new": 1, "own": 37, "page": 16,
         "heads": 32, "kv_heads": 8, "ragged": False},
        # 64 ragged prompts written into an fp8 cache and read back for a prefill that goes on.
        {"name": "kv_b64_fp8", "kind": "kv", "fmt": "fp8", "batch": 64, "new": 512, "own": 512, "page": 32,
         "heads": 32, "kv_heads": 8, "ragged": True},
        # One long prompt's last chunk into a bf16 cache that holds the chunks before it.
        {"name": "kv_b1_bf16_long", "kind": "kv", "fmt": "bf16", "batch": 1, "new": 4096, "own": 20011,
         "page": 128, "heads": 32, "kv_heads": 8, "ragged": False},
        # One sequence's next token over a short fp32 cache: latency.
        {"name": "attn_b1_f32", "kind": "attn", "fmt": "f32", "batch": 1, "new": 1, "own": 300, "prefix": 0,
         "page": 16, "heads": 32, "kv_heads": 8, "ragged": False},
        # A serving batch of unrelated, ragged sequences, one token each.
        {"name": "attn_b64_int8", "kind": "attn", "fmt": "int8", "batch": 64, "new": 1, "own": 2048,
         "prefix": 0, "page": 16, "heads": 32, "kv_heads": 8, "ragged": True},
        # The same batch behind one long system prompt.
        {"name": "attn_b64_fp8_prefix", "kind": "attn", "fmt": "fp8", "batch": 64, "new": 1, "own": 333,
         "prefix": 8192, "page": 64, "heads": 32, "kv_heads": 8, "ragged": True},
        # Four drafts and the token before them, ragged, behind a shared prompt.
        {"name": "attn_b16_int8_draft5", "kind": "attn", "fmt": "int8", "batch": 16, "new": 5, "own": 1000,
         "prefix": 2000, "page": 32, "heads": 32, "kv_heads": 8, "ragged": True},
        # A few very long contexts.
        {"name": "attn_b4_bf16_long", "kind": "attn", "fmt": "bf16", "batch": 4, "new": 1, "own": 65536,
         "prefix": 0, "page": 128, "heads": 32, "kv_heads": 8, "ragged": False},
        # One token's logits.
        {"name": "softmax_r1", "kind": "softmax", "rows": 1, "vocab": VOCAB, "temperature": 0.7},
        # The logits of 64 sequences' five positions.
        {"name": "softmax_r320", "kind": "softmax", "rows": 320, "vocab": VOCAB, "temperature": 1.0},
        # One sequence's four drafts.
        {"name": "verify_b1", "kind": "verify", "batch": 1, "drafts": 4, "vocab": VOCAB, "ragged": False},
        # A batch's, some with fewer drafts.
        {"name": "verify_b64", "kind": "verify", "batch": 64, "drafts": 4, "vocab": VOCAB, "ragged": True},
    ]


def _size(rng, lo, hi):
    """Spread over the logarithm of [lo, hi]."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["kv", "attn", "attn", "attn", "softmax", "verify"])
    if kind == "softmax":
        return {"kind": kind, "rows": _size(rng, 1, 320), "vocab": _size(rng, 500, VOCAB),
                "temperature": rng.choice([0.3, 0.7, 1.0, 1.5])}
    if kind == "verify":
        return {"kind": kind, "batch": _size(rng, 1, 64), "drafts": rng.randint(0, 8),
                "vocab": _size(rng, 500, VOCAB), "ragged": rng.random() < 0.5}
    fmt = rng.choice(FORMATS)
    heads, kv_heads = rng.choice([(32, 8), (32, 8), (32, 8), (16, 8), (8, 8), (16, 2)])
    c = {"kind": kind, "fmt": fmt, "batch": _size(rng, 1, 64), "page": rng.choice([16, 32, 64, 128]),
         "heads": heads, "kv_heads": kv_heads, "ragged": rng.random() < 0.6}
    if kind == "kv":
        most = max(1, 32768 // c["batch"])
        c["new"] = _size(rng, 1, min(4096, most))
        c["own"] = c["new"] + (_size(rng, 1, most) if rng.random() < 0.6 else 0)
    else:
        c["new"] = 1 if rng.random() < 0.5 else rng.randint(2, 8)
        c["own"] = max(c["new"], _size(rng, 1, (131072 if fmt in ("int8", "fp8") else 65536) // c["batch"]))
        c["prefix"] = _size(rng, 16, 8192) if rng.random() < 0.5 else 0
    return c


# -- inputs -------------------------------------------------------------------

class _Rng:
    """Seeded draws on the GPU; the same seed gives the same tensors."""

    def __init__(self, seed):
        self.g = torch.Generator(device="cuda")
        self.g.manual_seed(int(seed))

    def normal(self, *shape):
        return torch.randn(*shape, generator=self.g, device="cuda")

    def uniform(self, *shape):
        return torch.rand(*shape, generator=self.g, device="cuda")

    def order(self, n):
        return torch.randperm(n, generator=self.g, device="cuda").to(torch.int32)


def _lengths(case):
    """New tokens and own positions (new ones included) of each sequence."""
    B, new, most = case["batch"], case["new"], case["own"]
    if not case["ragged"]:
        return [new] * B, [most] * B
    n = [new - (5 * b % new) for b in range(B)]
    left = most - new
    return n, [n[b] + left - (left * (7 * b % B)) // (B + B // 4 + 1) for b in range(B)]


def _quantise(x, fmt):
    """Rows of 64 as the cache holds them: (stored values, fp32 scale or None)."""
    if fmt == "f32":
        return x, None
    if fmt == "bf16":
        return x.to(torch.bfloat16), None
    amax = x.abs().amax(-1)
    if fmt == "int8":
        s = (amax.double() / 127.0).float()
        q = torch.round(x.double() / s.double().unsqueeze(-1))  # in 64 bits: halves decide
        return torch.where(s.unsqueeze(-1) > 0, q, 0.0).clamp(-127, 127).to(torch.int8), s
    m, e = torch.frexp(amax.double() / E4M3_MAX)  # m in [0.5, 1): the power of two is 2^e, or 2^(e-1) for m = 0.5
    e = torch.where(m == 0.5, e - 1, e).clamp(min=-126)
    s = torch.ldexp(torch.ones_like(amax), e)
    return (x / s.unsqueeze(-1)).to(torch.float8_e4m3fn).view(torch.uint8), s


def _values(q, s, fmt):
    """The fp32 values that stored rows stand for."""
    if fmt == "f32":
        return q
    if fmt == "bf16":
        return q.float()
    q = q.float() if fmt == "int8" else q.view(torch.float8_e4m3fn).float()
    return q * s.unsqueeze(-1)


def _pool(r, case, pages):
    """k, v, k_scale, v_scale of a cache whose pages hold rows written earlier."""
    out = []
    for _ in range(2):
        x = r.normal(pages, case["kv_heads"], case["page"], HD)
        q, s = _quantise(x, case["fmt"])
        out.append((q.contiguous(), None if s is None else s.contiguous()))
    return out[0][0], out[1][0], out[0][1], out[1][1]


def _cache_inputs(case, seed):
    r, B, ps = _Rng(seed), case["batch"], case["page"]
    n, length = _lengths(case)
    prefix = case.get("prefix", 0)
    per_seq, shared = -(-max(length) // ps), -(-prefix // ps)
    total = B * per_seq + shared
    order = r.order(total)
    k, v, ks, vs = _pool(r, case, total)
    ld = (case["heads"] + 2 * case["kv_heads"]) * HD
    start = [0]
    for m in n:
        start.append(start[-1] + m)
    as_int = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
    return {"k": k, "v": v, "k_scale": ks, "v_scale": vs, "pages": order[:B * per_seq].view(B, per_seq).contiguous(),
            "prefix_pages": order[B * per_seq:].contiguous(), "own_len": as_int(length), "new_start": as_int(start),
            "qkv": r.normal(start[-1], ld), "ld": ld, "tokens": start[-1], "num_pages": total,
            "k_col": case["heads"] * HD, "v_col": (case["heads"] + case["kv_heads"]) * HD}


def _softmax_inputs(case, seed):
    return {"logits": _Rng(seed).normal(case["rows"], case["vocab"]) * 2.0}


def _verify_inputs(case, seed):
    """Target and draft probabilities of a draft that follows its target loosely, tokens drawn from the draft."""
    r, B, K, V = _Rng(seed), case["batch"], case["drafts"], case["vocab"]
    logits = r.normal(B, K + 1, V) * 2.0
    target = torch.softmax(logits, -1)
    draft = torch.softmax(logits[:, :K] + 0.7 * r.normal(B, K, V), -1)
    del logits
    c = draft.double().cumsum(-1)
    u = r.uniform(B, K).double().unsqueeze(-1) * c[..., -1:]
    ids = (c <= u).sum(-1).clamp(max=V - 1).to(torch.int32)
    n = [K - (b % (K + 1) if case["ragged"] else 0) for b in range(B)]
    return {"target": target.contiguous(), "draft": draft.contiguous(), "ids": ids.contiguous(),
            "n_valid": torch.tensor(n, dtype=torch.int32, device="cuda"), "u_accept": r.uniform(B, K),
            "u_sample": r.uniform(B)}


_INPUTS = {"kv": _cache_inputs, "attn": _cache_inputs, "softmax": _softmax_inputs, "verify": _verify_inputs}


# -- prepare and run ----------------------------------------------------------

def _p(t):
    return None if t is None else t.data_ptr()


def prepare(case, seed):
    kind = case["kind"]
    s = {"case": case, **_INPUTS[kind](case, seed)}
    if kind == "kv":
        rows = case["own"]
        s["k_out"], s["v_out"] = (torch.zeros(case["batch"] * rows, case["kv_heads"] * HD, device="cuda")
                                  for _ in range(2))
    elif kind == "attn":
        s["out"] = torch.zeros(s["tokens"], case["heads"] * HD, device="cuda")
    elif kind == "softmax":
        s["probs"] = torch.empty_like(s["logits"])
    else:
        s["accepted"] = torch.empty(case["batch"], dtype=torch.int32, device="cuda")
        s["out"] = torch.empty(case["batch"], case["drafts"] + 1, dtype=torch.int32, device="cuda")
    if own:
        from final_amd import lfm
        s["lfm"] = lfm
        need = 0
        if kind in ("kv", "attn"):
            fmt = {"f32": lfm.KV_F32, "bf16": lfm.KV_BF16, "int8": lfm.KV_INT8, "fp8": lfm.KV_FP8}[case["fmt"]]
            s["cache"] = lfm.KVCache(fmt, s["num_pages"], case["page"], _p(s["k"]), _p(s["v"]), _p(s["k_scale"]),
                                     _p(s["v_scale"]), kv_heads=case["kv_heads"])
            s["batch"] = lfm.KVBatch(case["batch"], _p(s["own_len"]), _p(s["pages"]), s["pages"].shape[1],
                                     max_new=case["new"], max_len=case["own"], tokens=s["tokens"],
                                     new_start=_p(s["new_start"]), prefix_pages=_p(s["prefix_pages"]),
                                     prefix_len=case.get("prefix", 0))
            if kind == "attn":
                need = lfm.kv_attention_workspace(s["cache"], s["batch"], heads=case["heads"])
        elif kind == "softmax":
            need = lfm.softmax_workspace(case["rows"], case["vocab"])
        else:
            need = lfm.verify_draft_workspace(case["batch"], case["vocab"])
        s["ws"], s["ws_bytes"] = torch.empty(max(need, 16), dtype=torch.uint8, device="cuda"), need
    torch.cuda.synchronize()
    return s


def _run_own(s):
    lfm, case, st = s["lfm"], s["case"], torch.cuda.current_stream().cuda_stream
    kind = case["kind"]
    if kind == "kv":
        lfm.kv_write(s["cache"], s["batch"], _p(s["qkv"]), s["ld"], heads=case["heads"], k_col=s["k_col"],
                     v_col=s["v_col"], stream=st)
        lfm.kv_read(s["cache"], s["batch"], _p(s["k_out"]), _p(s["v_out"]), case["own"], stream=st)
        return s["k_out"], s["v_out"]
    if kind == "attn":
        lfm.kv_attention(s["cache"], s["batch"], _p(s["qkv"]), s["ld"], _p(s["out"]), heads=case["heads"],
                         workspace=_p(s["ws"]), workspace_bytes=s["ws_bytes"], stream=st)
        return s["out"]
    if kind == "softmax":
        lfm.softmax(_p(s["logits"]), _p(s["probs"]), case["rows"], case["vocab"], temperature=case["temperature"],
                    workspace=_p(s["ws"]), workspace_bytes=s["ws_bytes"], stream=st)
        return s["probs"]
    lfm.verify_draft(_p(s["target"]), _p(s["draft"]), _p(s["ids"]), _p(s["u_accept"]), _p(s["u_sample"]),
                     _p(s["accepted"]), _p(s["out"]), case["batch"], case["drafts"], case["vocab"],
                     n_valid=_p(s["n_valid"]), workspace=_p(s["ws"]), workspace_bytes=s["ws_bytes"], stream=st)
    return s["accepted"], s["out"]


def _new_tokens(s):
    """Sequence, index among its new tokens and own position of each new token."""
    t = torch.arange(s["tokens"], device="cuda")
    b = torch.searchsorted(s["new_start"][1:].contiguous(), t, right=True)
    i = t - s["new_start"][b]
    n = s["new_start"][b + 1] - s["new_start"][b]
    return b, i, s["own_len"][b] - n + i


def _plain_kv(s):
    case, ps, H = s["case"], s["case"]["page"], s["case"]["kv_heads"]
    b, _, pos = _new_tokens(s)
    page, off = s["pages"][b, pos // ps].long(), pos % ps
    rows = torch.arange(case["own"], device="cuda")
    there = (rows < s["own_len"].unsqueeze(1)).view(case["batch"], -1, 1)
    at = s["pages"][:, (rows // ps).clamp(max=s["pages"].shape[1] - 1)].long()

    def one(store, scale, col, out):
        x = s["qkv"][:, col:col + H * HD].view(-1, H, HD)
        q, sc = _quantise(x, case["fmt"])
        store[page, :, off] = q
        if sc is not None:
            scale[page, :, off] = sc
        got = _values(store[at, :, rows % ps], None if sc is None else scale[at, :, rows % ps], case["fmt"])
        out.copy_(torch.where(there, got.reshape(case["batch"], -1, H * HD), out.view(case["batch"], -1, H * HD))
                  .view(out.shape))

    one(s["k"], s["k_scale"], s["k_col"], s["k_out"])
    one(s["v"], s["v_scale"], s["v_col"], s["v_out"])
    return s["k_out"], s["v_out"]


def _plain_attn(s):
    case, ps = s["case"], s["case"]["page"]
    B, N, KV, P = case["batch"], case["new"], case["kv_heads"], case["prefix"]
    G = case["heads"] // KV

    def rows_of(store, scale, table):
        """[sequences, kv head, position, 64] of the pages of a table."""
        x = _values(store[table.long()], None if scale is None else scale[table.long()], case["fmt"])
        return x.transpose(1, 2).reshape(table.shape[0], KV, -1, HD)

    # queries [B, kv head, new * group, 64], sequences with fewer padded by their last one
    n = s["new_start"][1:] - s["new_start"][:-1]
    i = torch.arange(N, device="cuda").expand(B, N)
    t = s["new_start"][:-1].unsqueeze(1) + torch.minimum(i, n.unsqueeze(1) - 1)
    q = s["qkv"][t.long(), :case["heads"] * HD].view(B, N, KV, G, HD).permute(0, 2, 1, 3, 4).reshape(B, KV, N * G, HD)
    q = q * 0.125
    k, v = rows_of(s["k"], s["k_scale"], s["pages"]), rows_of(s["v"], s["v_scale"], s["pages"])
    own_s = torch.matmul(q, k.transpose(2, 3).contiguous())
    last = s["own_len"].unsqueeze(1) - n.unsqueeze(1) + i  # the query's own position
    seen = torch.arange(k.shape[2], device="cuda") <= last.repeat_interleave(G, 1).unsqueeze(-1)
    scores = own_s.masked_fill(~seen.unsqueeze(1), -math.inf)
    if P:
        table = s["prefix_pages"].unsqueeze(0)
        kp, vp = (rows_of(a, c, table)[0, :, :P] for a, c in ((s["k"], s["k_scale"]), (s["v"], s["v_scale"])))
        qp = q.transpose(0, 1).reshape(KV, B * N * G, HD)
        sp = torch.matmul(qp, kp.transpose(1, 2).contiguous()).view(KV, B, N * G, P).transpose(0, 1)
        scores = torch.cat([scores, sp], -1)
    w = torch.exp(scores - scores.amax(-1, keepdim=True))
    w = w / w.sum(-1, keepdim=True)
    o = torch.matmul(w[..., :k.shape[2]], v)
    if P:
        wp = w[..., k.shape[2]:].transpose(0, 1).reshape(KV, B * N * G, P)
        o = o + torch.matmul(wp, vp.contiguous()).view(KV, B, N * G, HD).transpose(0, 1)
    o = o.view(B, KV, N, G, HD).permute(0, 2, 1, 3, 4).reshape(B, N, case["heads"] * HD)
    b, i, _ = _new_tokens(s)
    return o[b, i.long()]


def _plain_softmax(s):
    x = s["logits"]
    e = torch.exp((x - x.amax(-1, keepdim=True)) / s["case"]["temperature"])
    return e / e.sum(-1, keepdim=True)


def _plain_verify(s):
    case, B, K = s["case"], s["case"]["batch"], s["case"]["drafts"]
    n, seq = s["n_valid"], torch.arange(B, device="cuda")
    at = s["ids"].long().unsqueeze(-1)
    p = torch.gather(s["target"][:, :K], 2, at).squeeze(-1)
    q = torch.gather(s["draft"], 2, at).squeeze(-1)
    i = torch.arange(K, device="cuda")
    ok = (s["u_accept"].double() * q.double() < p.double()) & (i < n.unsqueeze(1))  # in 64 bits: a border
    a = ok.int().cumprod(1).sum(1)
    w = s["target"][seq, a].double()
    if K:
        less = s["draft"][seq, a.clamp(max=K - 1)].double()
        r = torch.where((a < n).unsqueeze(1), w - less, w).clamp(min=0)
        w = torch.where(r.sum(-1, keepdim=True) > 0, r, w)
    c = w.cumsum(-1)
    token = (c <= s["u_sample"].double().unsqueeze(1) * c[:, -1:]).sum(-1)
    token = torch.where(token < case["vocab"], token, -1).to(torch.int32)
    j = torch.arange(K + 1, device="cuda")
    ids = torch.cat([s["ids"], s["ids"].new_full((B, 1), -1)], 1)
    out = torch.where(j < a.unsqueeze(1), ids, torch.where(j == a.unsqueeze(1), token.unsqueeze(1), -1))
    return a.to(torch.int32), out.to(torch.int32)


_PLAIN = {"kv": _plain_kv, "attn": _plain_attn, "softmax": _plain_softmax, "verify": _plain_verify}


def run(state):
    return _run_own(state) if own else _PLAIN[state["case"]["kind"]](state)


# -- what a pass cannot do without ----------------------------------------------

def work(case):
    kind = case["kind"]
    if kind == "softmax":
        n = float(case["rows"]) * case["vocab"]
        return {"bytes": 8.0 * n, "flops": 4.0 * n}
    if kind == "verify":
        # one row of the target and one of the draft for each sequence, the draft's where there are drafts
        n = float(case["batch"]) * case["vocab"]
        return {"bytes": (8.0 if case["drafts"] else 4.0) * n, "flops": 3.0 * n}
    n, length = _lengths(case)
    per = {"f32": 4 * HD, "bf16": 2 * HD, "int8": HD + 4, "fp8": HD + 4}[case["fmt"]]  # a stored row
    KV, heads, tokens = case["kv_heads"], case["heads"], sum(n)
    if kind == "kv":
        row = 2.0 * KV * (per + 4 * HD)  # k and v, stored and in fp32
        return {"bytes": row * (tokens + sum(length)), "flops": 2.0 * KV * HD * 2 * (tokens + sum(length))}
    P = case["prefix"]
    pairs = sum(n[b] * (P + length[b]) - n[b] * (n[b] - 1) // 2 for b in range(case["batch"]))
    return {"bytes": 2.0 * KV * per * (sum(length) + P) + 2.0 * 4 * HD * heads * tokens,
            "flops": 4.0 * HD * heads * pairs}


# -- the same results in 64 bits -------------------------------------------------

def _e4m3(y):
    """y rounded to the nearest e4m3 value, halves to even (|y| <= 448)."""
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -20))).clamp(min=-6) - 3)
    return torch.round(y / step) * step


def _exact_stored(x, fmt):
    """The real values that rows x stand for once they are stored."""
    x = x.double()
    if fmt == "f32":
        return x
    if fmt == "bf16":
        step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=1e-30))) - 7)
        return torch.round(x / step) * step
    top = x.abs().amax(-1, keepdim=True)
    if fmt == "int8":
        s = (top / 127.0).float().double()  # the scale is an fp32 value
        return torch.round(x / s) * s
    s = torch.exp2(torch.ceil(torch.log2(top / 448.0)))
    return _e4m3(x / s) * s


def _exact_rows(d, case, which, table, count):
    """[position, kv head, 64] of the first `count` positions of a page table, as they are stored."""
    x, ps = d[which], case["page"]
    pos = torch.arange(count, device="cuda")
    page, off = table.long()[pos // ps], pos % ps
    x = x[page, :, off]
    if case["fmt"] in ("f32", "bf16"):
        return x.double()
    x = x.double() if case["fmt"] == "int8" else x.view(torch.float8_e4m3fn).float().double()
    return x * d[which + "_scale"][page, :, off].double().unsqueeze(-1)


def _exact_kv(case, seed):
    d = _cache_inputs(case, seed)
    n, length = _lengths(case)
    H, rows, outs = case["kv_heads"], case["own"], []
    for which, col in (("k", d["k_col"]), ("v", d["v_col"])):
        out = torch.zeros(case["batch"], rows, H * HD, dtype=torch.float64, device="cuda")
        new = _exact_stored(d["qkv"][:, col:col + H * HD].reshape(-1, H, HD), case["fmt"]).view(-1, H * HD)
        t = 0
        for b in range(case["batch"]):
            old = length[b] - n[b]
            if old:
                out[b, :old] = _exact_rows(d, case, which, d["pages"][b], old).view(old, -1)
            out[b, old:length[b]] = new[t:t + n[b]]
            t += n[b]
        outs.append(out.view(-1, H * HD))
    return tuple(outs)


def _exact_attn(case, seed):
    d = _cache_inputs(case, seed)
    n, length = _lengths(case)
    P, KV, heads = case["prefix"], case["kv_heads"], case["heads"]
    out = torch.empty(d["tokens"], heads, HD, dtype=torch.float64, device="cuda")
    front = [_exact_rows(d, case, w, d["prefix_pages"], P) for w in "kv"] if P else None
    t = 0
    for b in range(case["batch"]):
        k, v = (_exact_rows(d, case, w, d["pages"][b], length[b]) for w in "kv")
        if P:
            k, v = torch.cat([front[0], k]), torch.cat([front[1], v])
        for i in range(n[b]):
            end = P + length[b] - n[b] + i + 1
            q = d["qkv"][t, :heads * HD].double().view(KV, -1, HD)
            a = torch.stack([k[:end, g] @ q[g].t() for g in range(KV)], 1)
            a = torch.softmax(a / math.sqrt(HD), 0)
            out[t] = torch.stack([a[:, g].t() @ v[:end, g] for g in range(KV)]).view(heads, HD)
            t += 1
    return out.view(-1, heads * HD)


def _exact_verify(case, seed):
    d, K, V = _verify_inputs(case, seed), case["drafts"], case["vocab"]
    accepted, tokens = [], []
    for b in range(case["batch"]):
        n, a = int(d["n_valid"][b]), 0
        while a < n:
            x = int(d["ids"][b, a])
            if not float(d["u_accept"][b, a]) * float(d["draft"][b, a, x]) < float(d["target"][b, a, x]):
                break
            a += 1
        w = d["target"][b, a].double()
        if a < n:
            r = torch.relu(w - d["draft"][b, a].double())
            w = r if float(r.sum()) > 0 else w
        c = torch.cumsum(w, 0)
        above = torch.nonzero(c > float(d["u_sample"][b]) * c[V - 1])
        accepted.append(a)
        tokens.append([int(x) for x in d["ids"][b, :a]] + [int(above[0]) if len(above) else -1] + [-1] * (K - a))
    return (torch.tensor(accepted, dtype=torch.int32, device="cuda"),
            torch.tensor(tokens, dtype=torch.int32, device="cuda"))


def exact(case, seed):
    kind = case["kind"]
    if kind == "kv":
        return _exact_kv(case, seed)
    if kind == "attn":
        return _exact_attn(case, seed)
    if kind == "verify":
        return _exact_verify(case, seed)
    x = _softmax_inputs(case, seed)["logits"].double() / case["temperature"]
    return torch.exp(x - torch.logsumexp(x, -1, keepdim=True))
