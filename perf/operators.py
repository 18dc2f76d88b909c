"""The transformer-layer operators of the registry as cases that can be timed and checked.

Kinds of cases, each one call of a registered kernel:

  gemm       matrix product with bias, activation and a residual (or a gate) in its epilogue:
                 out = act(A W^T + bias) + other        or        act(A W^T + bias) * other
  norm       the norms after a block and before the next one, with the block's gate and the residual scale:
                 b' = N(block) * w0 (or block);   r = x + scale * gate * b';   y = N(r) * w1
             where N(v) = v / sqrt(mean(v^2) + eps)
  attention  softmax(scale * q k^T) v over packed sequences of different lengths, grouped heads; causal: the last
             query of a sequence sees its last key, a query without keys gives zeros

All tensors are bf16 (the bias fp32).  Activations are ~N(0,1), weights scaled as in the package's own workloads.
"""
import math

import torch

own = False

DEV = "cuda"
EPS = 1e-5

ACTS = ("none", "relu", "gelu", "gelu_tanh", "silu")


def listed():
    return [
        # Llama-3-8B output projection of a 512-token prompt, added to the residual stream
        dict(name="gemm_o_residual", kind="gemm", batch=1, m=512, n=4096, k=4096, act="none", bias=False, other="add"),
        # its down projection while decoding for 4 sequences: bound by the weights
        dict(name="gemm_down_decode", kind="gemm", batch=1, m=4, n=4096, k=14336, act="none", bias=False, other="add"),
        # its gate projection at prefill: SiLU, times the up projection
        dict(name="gemm_gate_prefill", kind="gemm", batch=1, m=4096, n=14336, k=4096, act="silu", bias=False, other="mul"),
        # a feed-forward layer with bias and GELU, odd everywhere
        dict(name="gemm_gelu_ragged", kind="gemm", batch=1, m=333, n=1000, k=712, act="gelu", bias=True, other="none"),
        # one token's residual add and norm in a 4096-wide layer: the launch itself counts
        dict(name="norm_token", kind="norm", rows=1, cols=4096, post=False, pre=True, gate="none", scale=1.0),
        # both norms of a 4096-wide layer at 512 tokens
        dict(name="norm_sandwich_512", kind="norm", rows=512, cols=4096, post=True, pre=True, gate="none", scale=1.0),
        # a long batch of wide rows, gated per column, residual scaled: bound by memory alone
        dict(name="norm_gated_long", kind="norm", rows=12007, cols=5120, post=True, pre=True, gate="cols", scale=0.22),
        # Llama-3-8B heads, one new token for each of 16 sequences with caches of very different lengths
        dict(name="attn_decode_ragged", kind="attention", q_lens="1," * 15 + "1",
             kv_lens="1,17,130,256,333,511,768,1025,1500,2048,2500,3001,3584,4000,4095,4096", heads=32, kv_heads=8, dim=128, causal=True),
        # one new token over one long cache: few rows, a long axis
        dict(name="attn_decode_long", kind="attention", q_lens="1", kv_lens="32768", heads=32, kv_heads=8, dim=128, causal=True),
        # GPT-2 heads, prompts of different lengths packed together
        dict(name="attn_packed_gpt2", kind="attention", q_lens="100,512,37,1024,1,640,333,901", kv_lens="100,512,37,1024,1,640,333,901",
             heads=12, kv_heads=12, dim=64, causal=True),
        # BERT-base: sixteen sequences seen in both directions, padding packed away
        dict(name="attn_bert_batch", kind="attention", q_lens="512,128,384,77,512,512,200,31,450,512,64,300,511,256,129,5",
             kv_lens="512,128,384,77,512,512,200,31,450,512,64,300,511,256,129,5", heads=12, kv_heads=12, dim=64, causal=False),
        # Llama-3-8B heads over a whole long prompt
        dict(name="attn_prefill_8k", kind="attention", q_lens="8192", kv_lens="8192", heads=32, kv_heads=8, dim=128, causal=True),
    ]


def _log(rng, lo, hi):
    """A whole number from lo to hi, spread evenly over the logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["gemm", "gemm", "norm", "attention", "attention"])
    if kind == "gemm":
        k, n = rng.choice([(4096, 4096), (4096, 1024), (4096, 14336), (14336, 4096), (768, 768), (1024, 4096), (2048, 2048), (712, 1000), (72, 136)])
        act, other = rng.choice(ACTS), rng.choice(["none", "add", "add", "mul"])
        batch = rng.choice([1, 1, 1, 3]) if k * n < 5_000_000 else 1
        return dict(kind=kind, batch=batch, m=_log(rng, 1, 4096), n=n, k=k, act=act, bias=rng.random() < 0.5, other=other)
    if kind == "norm":
        post, pre = rng.choice([(True, True), (True, True), (False, True), (True, False)])
        return dict(kind=kind, rows=_log(rng, 1, 12000), cols=rng.choice([64, 768, 1000, 1024, 2304, 4096, 5120, 8192]), post=post, pre=pre,
                    gate=rng.choice(["none", "cols", "rows"]), scale=rng.choice([1.0, 0.22, 0.5]))
    heads, kv_heads, dim = rng.choice([(32, 8, 128), (32, 8, 128), (12, 12, 64), (28, 4, 128), (16, 2, 64), (8, 1, 128), (24, 8, 80), (6, 3, 32)])
    form = rng.choice(["decode", "prompt", "prompt", "chunk"])
    seqs = _log(rng, 1, 48)
    if form == "decode":
        kv = [_log(rng, 1, 32768 // min(seqs, 8)) for _ in range(seqs)]
        q = [1] * seqs
    else:
        longest = int(8192 / math.sqrt(seqs))
        q = [_log(rng, 1, max(2, longest)) for _ in range(seqs)]
        kv = [n + _log(rng, 1, max(2, longest - n)) if form == "chunk" and longest - n > 2 else n for n in q]
    causal = form != "prompt" or rng.random() < 0.7
    return dict(kind=kind, q_lens=",".join(map(str, q)), kv_lens=",".join(map(str, kv)), heads=heads, kv_heads=kv_heads, dim=dim, causal=causal)


def _lens(case):
    return [int(x) for x in case["q_lens"].split(",")], [int(x) for x in case["kv_lens"].split(",")]


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)

    def randn(*shape, std=1.0, mean=0.0):
        x = torch.empty(shape, device=DEV, dtype=torch.bfloat16)
        return x.normal_(mean, std, generator=g)

    bf16 = dict(device=DEV, dtype=torch.bfloat16)
    st = {"case": case}
    if case["kind"] == "gemm":
        b, m, n, k = case["batch"], case["m"], case["n"], case["k"]
        st["a"], st["w"] = randn(b, m, k), randn(b, n, k, std=1.0 / math.sqrt(k))
        st["bias"] = torch.empty(n, device=DEV).normal_(0.0, 0.1, generator=g) if case["bias"] else None
        st["other"] = randn(b, m, n) if case["other"] != "none" else None
        st["out"] = torch.empty(b, m, n, **bf16)
    elif case["kind"] == "norm":
        rows, cols = case["rows"], case["cols"]
        st["x"], st["block"] = randn(rows, cols), randn(rows, cols, std=0.7)
        st["gate"] = {"none": lambda: None, "cols": lambda: randn(1, cols, std=0.5), "rows": lambda: randn(rows, cols, std=0.5)}[case["gate"]]()
        # the weights of the norms that are there, one row each: after the block, before the next
        st["w"] = randn(int(case["post"]) + int(case["pre"]), cols, std=0.1, mean=1.0)
        st["r"] = torch.empty(rows, cols, **bf16)
        st["y"] = torch.empty(rows, cols, **bf16) if case["pre"] else None
    else:
        ql, kl = _lens(case)
        heads, kvh, dim = case["heads"], case["kv_heads"], case["dim"]
        st["q"], st["k"], st["v"] = randn(sum(ql), heads, dim), randn(sum(kl), kvh, dim), randn(sum(kl), kvh, dim)
        cu = lambda lens: torch.tensor([0] + lens, device=DEV).cumsum(0).to(torch.int32)  # noqa: E731
        st["cu_q"], st["cu_kv"] = cu(ql), cu(kl)
        st["max_q"], st["max_kv"] = max(ql), max(kl)      # a program that packs its sequences knows the longest
        st["scale"] = 1.0 / math.sqrt(dim)
        st["out"] = torch.empty(sum(ql), heads, dim, **bf16)
    return st


# ------------------------------------------------------------------------------------------ plain forms

def _act(name, x):
    if name == "relu":
        return x.clamp(min=0)
    if name == "gelu":
        return 0.5 * x * (1 + torch.erf(x * math.sqrt(0.5)))
    if name == "gelu_tanh":
        return 0.5 * x * (1 + torch.tanh(math.sqrt(2 / math.pi) * (x + 0.044715 * x * x * x)))
    if name == "silu":
        return x / (1 + torch.exp(-x))
    return x


def _plain_gemm(st):
    c = st["case"]
    x = st["a"].float() @ st["w"].float().transpose(1, 2)
    if st["bias"] is not None:
        x = x + st["bias"]
    x = _act(c["act"], x)
    if c["other"] == "add":
        x = x + st["other"].float()
    elif c["other"] == "mul":
        x = x * st["other"].float()
    return {"out": x.to(torch.bfloat16)}


def _plain_norm(st):
    c = st["case"]
    w = st["w"].float()
    b = st["block"].float()
    if c["post"]:
        b = b / torch.sqrt((b * b).mean(-1, keepdim=True) + EPS) * w[0]
    if st["gate"] is not None:
        b = b * st["gate"].float()
    r = st["x"].float() + c["scale"] * b
    out = {"r": r.to(torch.bfloat16)}
    if c["pre"]:
        out["y"] = (r / torch.sqrt((r * r).mean(-1, keepdim=True) + EPS) * w[-1]).to(torch.bfloat16)
    return out


def _plain_attention(st):
    c = st["case"]
    heads, kvh, dim = c["heads"], c["kv_heads"], c["dim"]
    ql, kl = st["cu_q"][1:] - st["cu_q"][:-1], st["cu_kv"][1:] - st["cu_kv"][:-1]
    seqs, group = ql.numel(), heads // kvh
    iq, ik = torch.arange(st["max_q"], device=DEV), torch.arange(st["max_kv"], device=DEV)

    def padded(x, cu, idx):      # [seqs, longest, heads, dim] in 32 bits
        return x[(cu[:-1, None] + idx).clamp(max=x.shape[0] - 1)].float()

    q = padded(st["q"], st["cu_q"], iq).view(seqs, st["max_q"], kvh, group, dim).permute(0, 2, 3, 1, 4).reshape(seqs, kvh, group * st["max_q"], dim)
    k = padded(st["k"], st["cu_kv"], ik).permute(0, 2, 3, 1)
    v = padded(st["v"], st["cu_kv"], ik).permute(0, 2, 1, 3)
    seen = (ik < kl[:, None])[:, None, :].expand(seqs, st["max_q"], st["max_kv"])
    if c["causal"]:
        seen = seen & (ik <= (iq[:, None] + (kl - ql)[:, None, None]))
    s = (q @ k).mul_(st["scale"]).view(seqs, kvh, group, st["max_q"], st["max_kv"])
    s = s.masked_fill_(~seen[:, None, None], -math.inf)
    p = s.sub_(s.amax(-1, keepdim=True).clamp(min=-3e38)).exp_()
    total = p.sum(-1, keepdim=True)
    o = p.view(seqs, kvh, group * st["max_q"], st["max_kv"]) @ v
    o = o.view(seqs, kvh, group, st["max_q"], dim) / torch.where(total == 0, torch.ones_like(total), total)
    o = o.permute(0, 3, 1, 2, 4).reshape(seqs, st["max_q"], heads, dim)
    return {"out": o[iq < ql[:, None]].to(torch.bfloat16)}


# ------------------------------------------------------------------------------- the framework's kernels

_runtime = None


def _register(st):
    """The kernel of this program's buffers, registered once as the program would keep it."""
    global _runtime
    import bfuse_project_b200 as bf
    if _runtime is None:
        _runtime = bf.Runtime(0)
    rt, c = _runtime, st["case"]
    ptr = lambda name: None if st[name] is None else st[name].data_ptr()  # noqa: E731
    alone = bf.flag_share(1)
    if c["kind"] == "gemm":
        act = {"none": bf.ACT_NONE, "relu": bf.ACT_RELU, "gelu": bf.ACT_GELU, "gelu_tanh": bf.ACT_GELU_TANH, "silu": bf.ACT_SILU}[c["act"]]
        d = rt.describe("gemm_act", bf.OP_GEMM_ACT_BF16, (c["batch"], c["m"], c["n"], c["k"]), [ptr(n) for n in ("a", "w", "bias", "other", "out")],
                        flags=alone | bf.flag_act(act) | (bf.FLAG_MUL if c["other"] == "mul" else 0))
        outs = {"out": st["out"]}
    elif c["kind"] == "norm":
        norms = (bf.NORM_AFTER if c["post"] else 0) | (bf.NORM_BEFORE if c["pre"] else 0)
        d = rt.describe("residual_norm", bf.OP_RESIDUAL_NORM_BF16, (c["rows"], c["cols"], norms, 1 if c["gate"] == "rows" else 0),
                        [ptr(n) for n in ("x", "block", "gate", "w", "r", "y")], fparam=(EPS, c["scale"]), flags=alone)
        outs = {"r": st["r"], "y": st["y"]} if c["pre"] else {"r": st["r"]}
    else:
        shape = (st["cu_q"].numel() - 1, st["q"].shape[0], st["k"].shape[0], c["heads"], c["kv_heads"], c["dim"])
        d = rt.describe("attention", bf.OP_ATTENTION_BF16, shape, [ptr(n) for n in ("q", "k", "v", "cu_q", "cu_kv", "out")],
                        fparam=(st["scale"],), flags=alone | (bf.FLAG_CAUSAL if c["causal"] else 0))
        outs = {"out": st["out"]}
    return rt, rt.register_kernel(d), outs


def run(st):
    if own:
        if "kernel" not in st:
            st["kernel"] = _register(st)
        rt, kernel, outs = st["kernel"]
        rt.launch_kernel(kernel, torch.cuda.current_stream().cuda_stream)
        return outs
    return {"gemm": _plain_gemm, "norm": _plain_norm, "attention": _plain_attention}[st["case"]["kind"]](st)


# --------------------------------------------------------------------------------- work, and 64-bit values

def work(case):
    if case["kind"] == "gemm":
        b, m, n, k = case["batch"], case["m"], case["n"], case["k"]
        return {"bytes": 2 * b * (m * k + n * k + m * n * (1 if case["other"] == "none" else 2)) + (4 * n if case["bias"] else 0),
                "flops": 2 * b * m * n * k}
    if case["kind"] == "norm":
        rows, cols = case["rows"], case["cols"]
        tensors = 3 + int(case["pre"]) + (1 if case["gate"] == "rows" else 0)
        vectors = int(case["post"]) + int(case["pre"]) + (1 if case["gate"] == "cols" else 0)
        return {"bytes": 2 * cols * (rows * tensors + vectors), "flops": rows * cols * 10}
    ql, kl = _lens(case)
    pairs = 0
    for a, b in zip(ql, kl):
        if case["causal"]:      # query i sees max(0, b - a + i + 1) keys
            lo = max(0, a - b)
            pairs += (a - lo) * (b - a + lo + 1 + b) // 2 if a > lo else 0
        else:
            pairs += a * b
    return {"bytes": 4 * case["dim"] * (sum(ql) * case["heads"] + sum(kl) * case["kv_heads"]), "flops": 4 * case["dim"] * case["heads"] * pairs}


def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "gemm":
        outs = []
        for i in range(case["batch"]):
            z = torch.mm(st["a"][i].double(), st["w"][i].double().t())
            if st["bias"] is not None:
                z += st["bias"].double()[None, :]
            if case["act"] == "relu":
                z = torch.where(z > 0, z, torch.zeros_like(z))
            elif case["act"] == "gelu":
                z = z * torch.special.ndtr(z)
            elif case["act"] == "gelu_tanh":
                z = z * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))
            elif case["act"] == "silu":
                z = z * torch.sigmoid(z)
            if case["other"] == "add":
                z += st["other"][i].double()
            elif case["other"] == "mul":
                z *= st["other"][i].double()
            outs.append(z)
        return {"out": torch.stack(outs)}
    if case["kind"] == "norm":
        cols, w = case["cols"], st["w"].double()
        b = st["block"].double()
        if case["post"]:
            b = b * w[:1] * torch.rsqrt(b.pow(2).sum(1) / cols + EPS)[:, None]
        b = b * case["scale"]
        r = st["x"].double() + (b if st["gate"] is None else b * st["gate"].double())
        out = {"r": r}
        if case["pre"]:
            out["y"] = r * w[w.shape[0] - 1:] * torch.rsqrt(r.pow(2).sum(1) / cols + EPS)[:, None]
        return out
    ql, kl = _lens(case)
    group = case["heads"] // case["kv_heads"]
    out = torch.zeros(sum(ql), case["heads"], case["dim"], device=DEV, dtype=torch.float64)
    q0 = k0 = 0
    for a, b in zip(ql, kl):
        if b:
            for h in range(case["heads"]):
                q = st["q"][q0:q0 + a, h].double()
                k, v = st["k"][k0:k0 + b, h // group].double(), st["v"][k0:k0 + b, h // group].double()
                s = torch.mm(q, k.t()) * st["scale"]
                empty = None
                if case["causal"]:
                    hidden = torch.arange(b, device=DEV)[None, :] > torch.arange(b - a, b, device=DEV)[:, None]
                    s[hidden] = -math.inf
                    empty = hidden.all(1)
                o = torch.mm(torch.softmax(s, 1), v)
                if empty is not None:
                    o[empty] = 0.0
                out[q0:q0 + a, h] = o
        q0, k0 = q0 + a, k0 + b
    return {"out": out}
