"""The 4-bit block cache's operators as calls that can be timed and compared.

Keys and values are kept as E2M1 codes (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives) in
blocks of 64 positions, with one power of two as the scale of each 32 channels of a
position and KV head (K and V apart), and beside each position and KV head the attention
weight that it has had. A sequence is a row of block numbers; its newest positions are the
rows of the call. Five operators:

  rows     sp_hip_fp4_write, then sp_hip_fp4_read: K and V rows quantised into their blocks,
           and what they have become
  decode   sp_hip_fp4_attn_decode: one token's queries per sequence over its positions
  prefill  sp_hip_fp4_attn_prefill: several tokens' queries per sequence, causal
  weigh    sp_hip_fp4_weigh: the softmax weights of a call's queries added to the positions'
  evict    sp_hip_fp4_evict: each KV head keeps its first, its last and its heaviest positions

A scale is 2^e with the least e in [-40, 40] that holds the 32 channels' largest magnitude
within 6. A NaN is stored as 0 and what is past 6 * 2^40 at that number.
"""
import math
import os
import sys

import torch

own = False

DEV = "cuda"
BLOCK, GROUP = 64, 32
E_MIN, E_MAX = -40, 40
E2M1_MAX = 6.0
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _S():
    """The framework's binding (only where `own` is true)."""
    path = os.path.join(os.getcwd(), "shannon-prime-llama_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import sp_hip
    return sp_hip


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
# seqs sequences; ctx: positions of the longest after the call; new: rows of the longest
# in the call; ragged: lengths down to a quarter, at odd numbers; window: positions a
# query sees at most (0: all before it); keep, first, recent: positions that eviction
# leaves, and those of them that are kept whatever their weight.

def listed():
    return [
        # a decode step of 12 chats: one K and one V row per sequence appended to blocks that
        # are partly full, and read back as the cache holds them; latency counts
        dict(name="rows_step", op="rows", hd=128, heads=8, n_q=32, seqs=12, ctx=1000, new=1, ragged=True, dtype="f16"),
        # the prompts of six requests admitted together (the 1B-shaped model, head_dim 64)
        dict(name="rows_prompts", op="rows", hd=64, heads=8, n_q=32, seqs=6, ctx=4096, new=4096, ragged=True,
             dtype="f32"),
        # a short chat's decode step, where latency counts
        dict(name="decode_short", op="decode", hd=64, heads=8, n_q=32, seqs=1, ctx=777, new=1, ragged=False,
             dtype="f16", window=0, lse=False),
        # the 8B-shaped decode step at 32K, with the log-sum-exp that weighing needs
        dict(name="decode_32k", op="decode", hd=128, heads=8, n_q=32, seqs=1, ctx=32768, new=1, ragged=False,
             dtype="bf16", window=0, lse=True),
        # a serving step of the MHA, head_dim 96 model: 16 sequences of unequal length, float32 queries
        dict(name="decode_mha_batch", op="decode", hd=96, heads=32, n_q=32, seqs=16, ctx=4096, new=1, ragged=True,
             dtype="f32", window=0, lse=True),
        # five proposed tokens of each of 12 chats verified in one pass
        dict(name="verify_batch", op="prefill", hd=128, heads=8, n_q=32, seqs=12, ctx=4500, new=5, ragged=True,
             dtype="f16", window=0, lse=False),
        # a 2048-token chunk of the head_dim 256 model in a layer with a sliding window
        dict(name="prefill_window", op="prefill", hd=256, heads=8, n_q=16, seqs=1, ctx=9001, new=2048, ragged=False,
             dtype="bf16", window=1024, lse=False),
        # a 2048-token chunk of a 32K prompt, 8B-shaped: the largest
        dict(name="prefill_chunk", op="prefill", hd=128, heads=8, n_q=32, seqs=1, ctx=32768, new=2048, ragged=False,
             dtype="bf16", window=0, lse=True),
        # the weights of a decode step of 12 chats
        dict(name="weigh_step", op="weigh", hd=128, heads=8, n_q=32, seqs=12, ctx=4500, new=1, ragged=True,
             dtype="f16", window=0),
        # the last 64 tokens of a 32K prompt, whose weights say which of its positions stay
        dict(name="weigh_prompt", op="weigh", hd=128, heads=8, n_q=32, seqs=1, ctx=32768, new=64, ragged=False,
             dtype="bf16", window=0),
        # 12 chats that have passed their budget of 1000 positions by up to a block
        dict(name="evict_step", op="evict", hd=128, heads=8, n_q=32, seqs=12, ctx=1064, ragged=False, keep=1000,
             first=4, recent=128),
        # a 32K prompt cut to a quarter
        dict(name="evict_prompt", op="evict", hd=128, heads=8, n_q=32, seqs=1, ctx=32768, ragged=False, keep=8192,
             first=4, recent=512),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rows", "rows", "decode", "decode", "prefill", "prefill", "weigh", "weigh", "evict", "evict"])
    hd = rng.choice([64, 96, 128, 128, 256])
    heads = rng.choice([1, 2, 4, 8, 8, 32] if hd != 256 else [1, 4, 8])
    group = rng.choice([1, 2, 3, 4, 4, 8]) if heads < 32 else 1
    c = dict(op=op, hd=hd, heads=heads, n_q=heads * group, seqs=rng.choice([1, 1, 2, 3, 5, 12, 16, 40]))
    wide = heads * hd * c["seqs"]  # elements of a position of K
    if op == "evict":
        ctx = _log(rng, 2, max(64, min(131072, (1 << 27) // wide)))
        keep = _log(rng, 1, ctx)
        first = rng.choice([0, 0, min(4, keep)])
        return dict(c, ctx=ctx, ragged=rng.random() < 0.5, keep=keep, first=first,
                    recent=rng.choice([0, (keep - first) // 8, (keep - first) // 2, keep - first]))
    c["dtype"] = rng.choice(["f16", "bf16", "bf16", "f32"])
    if op == "rows":
        new = _log(rng, 1, max(2, min(32768, (1 << 25) // wide)))
        ctx = new + rng.choice([0, 0, 1, 63, 64, 500])
        return dict(c, ctx=ctx, new=new, ragged=rng.random() < 0.7)
    c["window"] = rng.choice([0, 0, 0, 100, 1024])
    if op == "decode":
        ctx = _log(rng, 1, max(64, min(131072, (1 << 28) // wide)))
        return dict(c, ctx=ctx, new=1, ragged=rng.random() < 0.7, lse=rng.random() < 0.4)
    if op == "prefill":
        new = _log(rng, 2, 2048)
        # new * ctx * seqs * n_q score elements, and ctx * seqs rows of K and V
        most = min((1 << 30) // (new * c["seqs"] * c["n_q"]), (1 << 27) // wide)
        c["lse"] = rng.random() < 0.4
    else:
        new = rng.choice([1, 1, 1, _log(rng, 2, 512)])
        most = min((1 << 28) // (new * c["seqs"] * c["n_q"]), (1 << 27) // wide)
    return dict(c, new=new, ctx=max(new, _log(rng, new, max(new + 1, min(65536, most)))), ragged=rng.random() < 0.7)


def _lengths(case):
    """Positions and rows of each sequence."""
    n, ctx, new = case["seqs"], case["ctx"], case.get("new", 1)
    if not case["ragged"]:
        return [ctx] * n, [new] * n
    cut = [((i * 5) % n) * 3 / (4 * n) for i in range(n)]
    lens = [max(1, ctx - int(c * ctx) - i) for i, c in enumerate(cut)]
    rows = [min(p, max(1, new - int(c * new) - (i if new > 8 * n else 0))) for i, (c, p) in enumerate(zip(cut, lens))]
    if new == ctx:
        rows = list(lens)
    return lens, rows


def _blocks(n):
    return (n + BLOCK - 1) // BLOCK


def work(case):
    lens, rows = _lengths(case)
    hd, H, n_q = case["hd"], case["heads"], case["n_q"]
    held = hd // 2 + hd // GROUP  # bytes of a row of one side and KV head
    if case["op"] == "evict":
        # what leaves its place: with weights that know nothing of the position, all but the first
        moved = sum(case["keep"] - case["first"] for p in lens if p > case["keep"])
        kept = sum(min(p, case["keep"]) for p in lens)
        seen = sum(p for p in lens if p > case["keep"])
        return {"bytes": float(H * (4 * seen + moved * 2 * (2 * held + 4) + 4 * kept)), "flops": float(H * seen)}
    esize = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "rows":
        n = sum(rows)
        return {"bytes": float(2 * n * H * 2 * (hd * esize + held) + 4 * n * H), "flops": float(8 * n * H * hd)}
    w = case["window"]
    seen = pairs = 0
    for p, r in zip(lens, rows):
        first = p - r
        seen += p if not w else p - max(0, first - w + 1)
        lo, hi = (first + 1, p) if not w else (min(first + 1, w), min(p, w))
        # rows see lo, lo+1, ... and w from there on
        ramp = hi - lo + 1
        pairs += (lo + hi) * ramp // 2 + (w * (r - ramp) if w else 0)
    queries = sum(rows) * n_q * (hd * esize + 4)
    if case["op"] == "weigh":
        return {"bytes": float(seen * H * (held + 8) + queries), "flops": float(2 * pairs * n_q * hd)}
    out = sum(rows) * n_q * (hd * esize * 2 + (4 if case["lse"] else 0))
    return {"bytes": float(seen * H * held * 2 + out), "flops": float(4 * pairs * n_q * hd)}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    return g


def _activations(g, n, heads, hd, dtype):
    """Rows [n, heads, hd] as a model's projections give them: unequal channels (log-normal),
    tokens of unequal strength, a few of them strong."""
    chan = torch.exp(0.5 * torch.randn((1, heads, hd), generator=g, device=DEV))
    x = torch.empty((n, heads, hd), dtype=dtype, device=DEV)
    for r0 in range(0, n, 1 << 16):
        m = min(1 << 16, n - r0)
        tok = torch.exp(0.3 * torch.randn((m, 1, 1), generator=g, device=DEV))
        tok = torch.where(torch.rand((m, 1, 1), generator=g, device=DEV) < 0.01, tok * 8, tok)
        x[r0:r0 + m] = (torch.randn((m, heads, hd), generator=g, device=DEV) * chan * tok).to(dtype)
    return x


def _inputs(case, seed):
    """Everything a call reads, in tensors: the cache's codes, scales and weights (layer 0 of
    one layer), the table of blocks, lengths and first rows, and the rows."""
    lens, rows = _lengths(case)
    hd, H, n_q, n = case["hd"], case["heads"], case["n_q"], case["seqs"]
    g = _gen(seed * 7919 + 17)
    used = [_blocks(p) for p in lens]
    stride, n_blocks = max(used), sum(used) + 3
    at = torch.randperm(n_blocks, generator=g, device=DEV)[:sum(used)].to(torch.int32)
    table = torch.full((n, stride), -1, dtype=torch.int32, device=DEV)
    starts = [sum(used[:i]) for i in range(n)]
    for i in range(n):
        table[i, :used[i]] = at[starts[i]:starts[i] + used[i]]
    row = [0]
    for r in rows:
        row.append(row[-1] + r)
    s = dict(case=case, lens=lens, rows=rows, table=table, n_blocks=n_blocks,
             d_len=torch.tensor(lens, dtype=torch.int32, device=DEV),
             d_row=torch.tensor(row, dtype=torch.int32, device=DEV) if case.get("new", 1) > 1 else None,
             n_rows=row[-1])
    codes = []
    for _ in range(2):  # what the blocks hold before the call
        k = torch.empty((1, n_blocks, H, 32 * hd), dtype=torch.uint8, device=DEV)
        e = torch.empty((1, n_blocks, H, hd // GROUP * BLOCK), dtype=torch.uint8, device=DEV)
        step = max(1, (1 << 26) // (BLOCK * H * hd))
        for b0 in range(0, n_blocks, step):
            m = min(step, n_blocks - b0)
            k[0, b0:b0 + m], e[0, b0:b0 + m] = _pack(*_encode(
                _activations(g, m * BLOCK, H, hd, torch.float32).view(m, BLOCK, H, hd)))
        codes += [k, e]
    s["k"], s["k_exp"], s["v"], s["v_exp"] = codes
    # of the steps before: most positions had little, a few much
    s["weight"] = torch.exp(2.0 * torch.randn((1, n_blocks, H, BLOCK), generator=g, device=DEV)) / case["ctx"]
    if case["op"] == "evict":
        return s
    dt = DTYPES[case["dtype"]]
    if case["op"] == "rows":
        s["k_rows"] = _activations(g, row[-1], H, hd, dt)
        s["v_rows"] = _activations(g, row[-1], H, hd, dt)
        return s
    s["q"] = _activations(g, row[-1], n_q, hd, dt)
    s["scale"] = 1.0 / math.sqrt(hd)
    if case["op"] == "weigh":  # what the attention call has returned
        top, total, _, _ = _scores(s)
        s["lse"] = _to_rows(s, (top + total.log()).squeeze(-1)).contiguous()
    return s


class _Memory:
    """Device memory that a cache owns, as torch can take it without a copy: the tensor holds
    this object, and this object the cache."""

    def __init__(self, cache, ptr, shape, kind):
        self.cache = cache
        self.__cuda_array_interface__ = dict(shape=tuple(shape), typestr=kind, data=(int(ptr), False), version=2)


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:  # the cache is the library's: the same contents, held in its memory
        S = _S()
        cfg = S.config(case["hd"], 1, case["heads"])
        s["cache"] = S.Fp4Cache(cfg, s["n_blocks"], torch.cuda.current_stream().cuda_stream)
        c = s["cache"].c
        for name, ptr in (("k", c.d_k_codes), ("k_exp", c.d_k_exp), ("v", c.d_v_codes), ("v_exp", c.d_v_exp),
                          ("weight", c.d_weight)):
            kind = "<f4" if name == "weight" else "|u1"
            mine = torch.as_tensor(_Memory(s["cache"], ptr, s[name].shape, kind), device="cuda")
            mine.copy_(s[name])
            s[name] = mine
        s["batch"] = S.Fp4Batch(case["seqs"], s["table"].shape[1], s["table"].data_ptr(), s["d_len"].data_ptr(),
                                s["d_row"].data_ptr() if s["d_row"] is not None else 0, s["n_rows"])
    return s


# ---------------------------------------------------------------------------
# the framework's calls
# ---------------------------------------------------------------------------

def _own(s):
    S, case = _S(), s["case"]
    L, op, hd, H, n_q = S.lib(), case["op"], case["hd"], case["heads"], case["n_q"]
    stream = torch.cuda.current_stream().cuda_stream
    cache, batch = s["cache"].ref, s["batch"].ref
    if op == "evict":
        kept = torch.empty((case["seqs"], H, case["keep"]), dtype=torch.int32, device="cuda")
        S.check(L.sp_hip_fp4_evict(cache, 0, batch, case["keep"], case["first"], case["recent"], kept.data_ptr(),
                                   stream), "sp_hip_fp4_evict")
        return _held(s, kept)
    code, dt = {"f32": S.DTYPE_F32, "f16": S.DTYPE_F16, "bf16": S.DTYPE_BF16}[case["dtype"]], DTYPES[case["dtype"]]
    if op == "rows":
        S.check(L.sp_hip_fp4_write(cache, 0, batch, s["k_rows"].data_ptr(), s["v_rows"].data_ptr(), H * hd, code,
                                   stream), "sp_hip_fp4_write")
        k, v = (torch.empty((s["n_rows"], H, hd), dtype=dt, device="cuda") for _ in range(2))
        S.check(L.sp_hip_fp4_read(cache, 0, batch, k.data_ptr(), v.data_ptr(), H * hd, code, stream),
                "sp_hip_fp4_read")
        return {"k": k, "v": v, "weight": s["weight"]}
    if op == "weigh":
        S.check(L.sp_hip_fp4_weigh(cache, 0, batch, s["q"].data_ptr(), n_q * hd, n_q, code, s["scale"],
                                   case["window"], s["lse"].data_ptr(), stream), "sp_hip_fp4_weigh")
        return {"weight": s["weight"]}
    out = torch.empty((s["n_rows"], n_q, hd), dtype=dt, device="cuda")
    lse = torch.empty((s["n_rows"], n_q), dtype=torch.float32, device="cuda") if case["lse"] else None
    call = L.sp_hip_fp4_attn_decode if op == "decode" else L.sp_hip_fp4_attn_prefill
    S.check(call(cache, 0, batch, s["q"].data_ptr(), n_q * hd, n_q, code, s["scale"], case["window"], out.data_ptr(),
                 n_q * hd, lse.data_ptr() if lse is not None else None, stream), "sp_hip_fp4_attn")
    return {"out": out, "lse": lse}


def _held(s, kept):
    """What eviction leaves. Codes and scales are the cache's bytes: rows are moved, nothing
    of them is computed."""
    return {"kept": kept, "weight": s["weight"], "k": s["k"], "k_exp": s["k_exp"], "v": s["v"], "v_exp": s["v_exp"]}


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------
# A block's codes lie in planes of eight channels, [heads, hd / 8, 64 positions], four bytes a
# position with the lowest channel in the lowest four bits. Its scales lie in planes of 32
# channels; in one, position p has byte (p // 4 % 4) * 16 + p // 16 * 4 + p % 4.

def _pow2(e):
    return ((e + 127) << 23).view(torch.float32)


def _encode(x):
    """Rows [..., hd] in float32: codes [..., hd] (sign, then the number's index) and biased
    exponents [..., hd / 32]."""
    x = torch.where(torch.isnan(x), 0.0, x).clamp(-E2M1_MAX * 2.0 ** E_MAX, E2M1_MAX * 2.0 ** E_MAX)
    g = x.unflatten(-1, (-1, GROUP))
    # 6 = 1.5 * 2^2: one more than floor(log2(amax)) - 2 where the fraction is past 1.5
    e = (((g.abs().amax(-1).view(torch.int32) + 0x3FFFFF) >> 23) - 129).clamp(E_MIN, E_MAX)
    y = g * _pow2(-e)[..., None]
    a = y.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    a = torch.round(a / step) * step
    code = torch.where(a < 2, a * 2, torch.where(a < 4, a + 2, a * 0.5 + 4)).to(torch.uint8)
    return (code + 8 * torch.signbit(y).to(torch.uint8)).flatten(-2), (e + 127).to(torch.uint8)


def _pack(code, e):
    """[blocks, 64, H, hd] and [blocks, 64, H, hd / 32] -> the order blocks are held in."""
    b, _, H, hd = code.shape
    two = code[..., 0::2] + 16 * code[..., 1::2]
    k = two.view(b, BLOCK, H, hd // 8, 4).permute(0, 2, 3, 1, 4).reshape(b, H, -1)
    return k, e.view(b, 4, 4, 4, H, -1).permute(0, 4, 5, 2, 1, 3).reshape(b, H, -1)


def _values(s, side, blocks):
    """What the listed blocks hold: [len(blocks), 64, H, hd] in float32."""
    hd, H = s["case"]["hd"], s["case"]["heads"]
    codes, exps = (s["k"], s["k_exp"]) if side == 0 else (s["v"], s["v_exp"])
    b = blocks.numel()
    two = codes[0][blocks].view(b, H, hd // 8, BLOCK, 4).permute(0, 3, 1, 2, 4).reshape(b, BLOCK, H, hd // 2)
    c = torch.stack((two & 15, two >> 4), -1).reshape(b, BLOCK, H, hd)
    i = (c & 7).float()
    a = torch.where(i < 4, i * 0.5, torch.where(i < 6, i - 2, i * 2 - 8))
    e = exps[0][blocks].view(b, H, hd // GROUP, 4, 4, 4).permute(0, 4, 3, 5, 1, 2).reshape(b, BLOCK, H, hd // GROUP)
    return torch.where(c > 7, -a, a) * _pow2(e.int() - 127).repeat_interleave(GROUP, -1)


def _row_places(s):
    """Of every row of the call: its sequence and its position."""
    first = torch.zeros(s["case"]["seqs"] + 1, dtype=torch.int64, device=DEV)
    n = torch.arange(s["n_rows"], device=DEV)
    first[1:] = n[:s["case"]["seqs"]] + 1 if s["d_row"] is None else s["d_row"][1:]
    seq = torch.searchsorted(first[1:], n, right=True)
    return seq, s["d_len"].long()[seq] - (first[1:][seq] - n), first


def _exp_place(p):
    return p // 4 % 4 * 16 + p // 16 * 4 + p % 4


def _plain_rows(s):
    hd, H = s["case"]["hd"], s["case"]["heads"]
    seq, pos, _ = _row_places(s)
    block, at = s["table"].long()[seq, pos // BLOCK], pos % BLOCK
    # a block whose first position is written starts anew: what lies behind its rows has the least scale
    anew = block[at == 0]
    got = {}
    for name in "kv":
        code, e = _encode(s[name + "_rows"].float())
        planes = s[name].view(-1, H, hd // 8, BLOCK, 4)
        exps = s[name + "_exp"].view(-1, H, hd // GROUP, BLOCK)
        exps[anew] = 127 + E_MIN
        planes[block, :, :, at] = (code[..., 0::2] + 16 * code[..., 1::2]).view(-1, H, hd // 8, 4)
        exps[block, :, :, _exp_place(at)] = e
        touched, which = torch.unique(block, return_inverse=True)
        got[name] = _values(s, "kv".index(name), touched)[which, at].to(DTYPES[s["case"]["dtype"]])
    s["weight"][0][block, :, at] = 0.0
    return dict(got, weight=s["weight"])


def _scores(s):
    """Largest score and sum of each row of queries, the exponentials, and V, padded to the
    longest sequence: [n, H, R, group, .]."""
    case = s["case"]
    n, H, hd, n_q = case["seqs"], case["heads"], case["hd"], case["n_q"]
    group = n_q // H
    seq, pos, first = _row_places(s)
    R, Lk = max(s["rows"]), s["table"].shape[1] * BLOCK
    flat = s["table"].long().clamp(min=0).view(-1)
    K, V = (_values(s, side, flat).view(n, Lk, H, hd).permute(0, 2, 1, 3) for side in range(2))
    # queries padded to [n, R] rows, the heads of a group beside each other
    at = torch.arange(s["n_rows"], device=DEV) - first[:-1][seq]
    q = torch.zeros((n, R, H, group, hd), dtype=torch.float32, device=DEV)
    q[seq, at] = s["q"].float().view(-1, H, group, hd)
    q = q.permute(0, 2, 1, 3, 4).reshape(n, H, R * group, hd)
    place = torch.full((n, R), -1, dtype=torch.int64, device=DEV)
    place[seq, at] = pos
    key = torch.arange(Lk, device=DEV)
    sees = key[None, None, :] <= place[:, :, None]
    if case["window"]:
        sees &= key[None, None, :] > place[:, :, None] - case["window"]
    hidden = ~sees[:, None, :, None, :]
    sc = torch.matmul(q, K.transpose(-1, -2).contiguous()).mul_(s["scale"]).view(n, H, R, group, Lk)
    sc.masked_fill_(hidden, -math.inf)
    top = sc.amax(-1, keepdim=True)
    p = sc.sub_(torch.where(torch.isinf(top), 0.0, top)).exp_()
    return top, p.sum(-1, keepdim=True), p, V


def _to_rows(s, x):
    """[n, H, R, group, ...] -> the call's rows, [n_rows, n_q, ...]."""
    n, n_q = s["case"]["seqs"], s["case"]["n_q"]
    seq, _, first = _row_places(s)
    at = torch.arange(s["n_rows"], device=DEV) - first[:-1][seq]
    x = x.transpose(1, 2)
    return x.reshape((n, x.shape[1], n_q) + x.shape[4:])[seq, at]


def _plain_attn(s):
    top, total, p, V = _scores(s)
    n, H, R, group, Lk = p.shape
    out = torch.matmul(p.view(n, H, R * group, Lk), V.contiguous()).view(n, H, R, group, -1)
    out = _to_rows(s, torch.where(total > 0, out / total, 0.0)).to(DTYPES[s["case"]["dtype"]])
    return {"out": out, "lse": _to_rows(s, (top + total.log()).squeeze(-1)) if s["case"]["lse"] else None}


def _plain_weigh(s):
    case = s["case"]
    n, H, group = case["seqs"], case["heads"], case["n_q"] // case["heads"]
    top, _, p, _ = _scores(s)
    seq, _, first = _row_places(s)
    at = torch.arange(s["n_rows"], device=DEV) - first[:-1][seq]
    lse = torch.full((n, p.shape[2], H, group), math.inf, device=DEV)
    lse[seq, at] = s["lse"].view(-1, H, group)
    lse = lse.transpose(1, 2)[..., None]
    w = p.mul_(torch.exp(torch.where(torch.isinf(top), 0.0, top) - lse)).sum((2, 3))    # [n, H, Lk]
    used = s["table"] >= 0
    add = w.view(n, H, -1, BLOCK).transpose(1, 2)[used]
    s["weight"][0][s["table"].long()[used]] += add
    return {"weight": s["weight"]}


def _plain_evict(s):
    case = s["case"]
    n, H, hd, keep = case["seqs"], case["heads"], case["hd"], case["keep"]
    length = s["d_len"].long()[:, None, None]
    flat = s["table"].long().clamp(min=0)
    w = s["weight"][0][flat].permute(0, 2, 1, 3).reshape(n, H, -1)
    t = torch.arange(w.shape[-1], device=DEV)
    w = torch.where((t < case["first"]) | (t >= length - case["recent"]), math.inf, w)
    w = torch.where(t < length, w, -math.inf)
    pad = max(0, keep - w.shape[-1])
    w = torch.nn.functional.pad(w, (0, pad), value=-math.inf)
    old = torch.sort(w, dim=-1, descending=True, stable=True)[1][..., :keep].sort(-1)[0]
    kept = torch.where(old < length, old, -1).to(torch.int32)
    # rows that leave their place, of sequences that are cut
    cut = (length > keep) & (old != torch.arange(keep, device=DEV))
    i, h, j = torch.nonzero(cut, as_tuple=True)
    p = old[i, h, j]
    src, dst = flat[i, p // BLOCK], flat[i, j // BLOCK]
    end = torch.nonzero((s["d_len"] > keep) & (keep % BLOCK > 0)).view(-1)
    behind = _exp_place(torch.arange(keep % BLOCK, BLOCK, device=DEV))
    for name in "kv":
        planes = s[name].view(-1, H, hd // 8, BLOCK, 4)
        planes[dst, h, :, j % BLOCK] = planes[src, h, :, p % BLOCK]
        exps = s[name + "_exp"].view(-1, H, hd // GROUP, BLOCK)
        exps[dst, h, :, _exp_place(j % BLOCK)] = exps[src, h, :, _exp_place(p % BLOCK)]
        exps.transpose(0, 3)[behind[:, None], :, :, flat[end, keep // BLOCK].view(1, -1)] = 127 + E_MIN
    s["weight"][0][dst, h, j % BLOCK] = s["weight"][0][src, h, p % BLOCK]
    return _held(s, kept)


def run(s):
    if own:
        return _own(s)
    op = s["case"]["op"]
    if op == "rows":
        return _plain_rows(s)
    if op == "weigh":
        return _plain_weigh(s)
    return _plain_evict(s) if op == "evict" else _plain_attn(s)


# ---------------------------------------------------------------------------
# 64 bits
# ---------------------------------------------------------------------------

_NUMBERS = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def _nearest(y):
    """The E2M1 number nearest to y, by comparison with the borders between two of them (a
    border itself goes to the number with the even index), past 6 that."""
    a, r = y.abs(), torch.zeros_like(y)
    for i in range(7):
        mid = (_NUMBERS[i] + _NUMBERS[i + 1]) / 2
        r = torch.where(a > mid if i % 2 == 0 else a >= mid, _NUMBERS[i + 1], r)
    return torch.where(y < 0, -r, r)


def _least_exponent(amax):
    """By comparison, from below."""
    e = torch.full(amax.shape, float(E_MIN), dtype=torch.float64, device=DEV)
    for k in range(E_MIN, E_MAX):
        e = torch.where(amax > E2M1_MAX * 2.0 ** k, float(k + 1), e)
    return e


def _held64(s, side, blocks, h, hd):
    """Positions [64 * len(blocks), hd] of one KV head, element by element."""
    codes, exps = ((s["k"], s["k_exp"]), (s["v"], s["v_exp"]))[side]
    t = torch.arange(BLOCK, device=DEV)[:, None]
    d = torch.arange(hd, device=DEV)[None, :]
    byte = ((d // 8) * BLOCK + t) * 4 + d % 8 // 2
    c = (codes[0][blocks, h][:, byte].long() >> (4 * (d % 2))) & 15
    numbers = torch.tensor(_NUMBERS + [-x for x in _NUMBERS], dtype=torch.float64, device=DEV)
    e = exps[0][blocks, h][:, d // GROUP * BLOCK + (t // 4 % 4) * 16 + t // 16 * 4 + t % 4]
    return (numbers[c] * torch.exp2(e.double() - 127)).view(-1, hd)


def exact(case, seed):
    s = _inputs(case, seed)
    hd, H, n, op = case["hd"], case["heads"], case["seqs"], case["op"]
    table = s["table"].cpu().tolist()
    weight = s["weight"].double()
    if op == "rows":
        got = {}
        for name in "kv":
            x = s[name + "_rows"].double().view(-1, H, hd // GROUP, GROUP)
            e = torch.exp2(_least_exponent(x.abs().amax(-1, keepdim=True)))
            got[name] = (_nearest(x / e) * e).view(-1, H, hd)
        for i in range(n):
            for p in range(s["lens"][i] - s["rows"][i], s["lens"][i]):
                weight[0, table[i][p // BLOCK], :, p % BLOCK] = 0.0
        return dict(got, weight=weight)
    if op == "evict":
        keep = case["keep"]
        for i in range(n):
            p = s["lens"][i]
            if p <= keep:
                continue
            blocks = torch.tensor(table[i][:_blocks(p)], device=DEV)
            for h in range(H):
                w = weight[0, blocks, h].reshape(-1)[:p]
                inner = w[case["first"]:p - case["recent"]]
                # heavier ones, and equal ones before: whose number is below the count that stays
                order = torch.argsort(inner, descending=True, stable=True)
                stays = torch.ones(p, dtype=torch.bool, device=DEV)
                stays[case["first"] + order[keep - case["first"] - case["recent"]:]] = False
                to = torch.arange(keep, device=DEV)
                weight[0, blocks[to // BLOCK], h, to % BLOCK] = w[stays].clone()
        return {"kept": None, "weight": weight, "k": None, "k_exp": None, "v": None, "v_exp": None}
    n_q, w = case["n_q"], case["window"]
    group = n_q // H
    outs, lses, r0 = [], [], 0
    for i in range(n):
        p, r = s["lens"][i], s["rows"][i]
        j0 = max(0, p - r - w + 1) // BLOCK if w else 0
        blocks = torch.tensor(table[i][j0:_blocks(p)], device=DEV)
        q = s["q"][r0:r0 + r].double()
        out = torch.empty((r, n_q, hd), dtype=torch.float64, device=DEV)
        lse = torch.empty((r, n_q), dtype=torch.float64, device=DEV)
        key = torch.arange(j0 * BLOCK, p, device=DEV)
        place = torch.arange(p - r, p, device=DEV)
        hide = key[None] > place[:, None]
        if w:
            hide |= key[None] <= place[:, None] - w
        for h in range(H):
            K = _held64(s, 0, blocks, h, hd)[:p - j0 * BLOCK]
            V = _held64(s, 1, blocks, h, hd)[:p - j0 * BLOCK] if op != "weigh" else None
            for gq in range(h * group, (h + 1) * group):
                sc = (q[:, gq] @ K.T) * s["scale"]
                sc.masked_fill_(hide, -math.inf)
                if op == "weigh":
                    add = torch.exp(sc - s["lse"][r0:r0 + r, gq, None].double()).sum(0)
                    add = torch.nn.functional.pad(add, (0, blocks.numel() * BLOCK - add.numel()))
                    weight[0, blocks, h] += add.view(-1, BLOCK)
                    continue
                lse[:, gq] = torch.logsumexp(sc, -1)
                out[:, gq] = torch.exp(sc - lse[:, gq, None]) @ V
        outs.append(out)
        lses.append(lse)
        r0 += r
    if op == "weigh":
        return {"weight": weight}
    return {"out": torch.cat(outs), "lse": torch.cat(lses) if case["lse"] else None}
