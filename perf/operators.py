"""What is timed of the packed-sequence attention and of the distillation from a teacher's top logits.

Three operators, each in a plain form (elementary torch operations in 32 bits) and through the package's entry points:

  attention   ops.packed_attention         queries of many sequences laid end to end, grouped heads, forward or forward + backward
  top         ops.top_logits               the k largest logits of each row with their classes, and the row's log-sum-exp
  distil      ops.soft_cross_entropy_top   the distillation loss from such top logits and the gradient of the student's logits

A case holds plain values only; the sequences' lengths are a function of the case, everything else of the seed (k_max = 0: as
many keys as queries).
"""
import math
import random

import torch

own = False

VOCAB = 30522                     # the text encoder's vocabulary


# ---------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------
def listed():
    return [
        # one answer token for each of 24 questions, right behind a short prompt: latency is all there is to it
        dict(name="step_short", op="attention", dtype="bf16", seqs=24, q_min=1, q_max=1, k_min=6, k_max=40, heads=12, kv_heads=12,
             dim=64, causal=True, slots=True, train=False),
        # one token for each of 12 sequences against long caches that are only partly filled
        dict(name="step_long", op="attention", dtype="bf16", seqs=12, q_min=1, q_max=1, k_min=6000, k_max=40000, heads=32, kv_heads=8,
             dim=128, causal=True, slots=True, train=False),
        # the answers of a VQA batch, packed: very many, very short sequences, one training pass of one decoder layer
        dict(name="answers_train", op="attention", dtype="bf16", seqs=300, q_min=3, q_max=16, k_min=0, k_max=0, heads=12, kv_heads=12,
             dim=64, causal=True, slots=False, train=True),
        # captions and paragraphs, packed, few key heads: an ordinary training pass
        dict(name="texts_train", op="attention", dtype="bf16", seqs=20, q_min=40, q_max=900, k_min=0, k_max=0, heads=12, kv_heads=4,
             dim=64, causal=True, slots=False, train=True),
        # whole prompts of a serving batch
        dict(name="prompts", op="attention", dtype="bf16", seqs=6, q_min=1500, q_max=9000, k_min=0, k_max=0, heads=32, kv_heads=8,
             dim=128, causal=True, slots=False, train=False),
        # long documents, training
        dict(name="documents_train", op="attention", dtype="bf16", seqs=5, q_min=1000, q_max=5000, k_min=0, k_max=0, heads=16, kv_heads=4,
             dim=128, causal=True, slots=False, train=True),
        # questions attending to packed encoder states of other lengths, 32-bit parity path
        dict(name="cross_f32_train", op="attention", dtype="f32", seqs=9, q_min=5, q_max=90, k_min=20, k_max=400, heads=12, kv_heads=12,
             dim=64, causal=False, slots=False, train=True),
        # the top classes of one decoding step
        dict(name="top_step", op="top", dtype="bf16", rows=7, classes=VOCAB, k=16, temperature=1.0, padded=True),
        # a teacher's masked-token rows of a large batch, kept as top logits instead of whole rows
        dict(name="top_teacher", op="top", dtype="bf16", rows=3000, classes=VOCAB, k=64, temperature=2.0, padded=True),
        # the answer tokens of a VQA batch with the answers' weights, target renormalised over the kept classes
        dict(name="distil_answers", op="distil", dtype="bf16", rows=330, classes=VOCAB, k=16, temperature=1.0, padded=True,
             rest=False, weighted=True),
        # the masked-token rows of a large batch, with the teacher's remaining mass as one more class
        dict(name="distil_teacher", op="distil", dtype="bf16", rows=5000, classes=VOCAB, k=64, temperature=2.0, padded=True,
             rest=True, weighted=False),
        # the 32-bit parity path on unpadded rows
        dict(name="distil_f32", op="distil", dtype="f32", rows=77, classes=VOCAB, k=32, temperature=1.5, padded=False,
             rest=True, weighted=True),
    ]


def _spread(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["attention", "attention", "attention", "top", "distil"])
    dtype = rng.choice(["bf16", "bf16", "bf16", "f32"])
    if op != "attention":
        rows = _spread(rng, 1, 3000 if dtype == "bf16" else 800)
        case = dict(op=op, dtype=dtype, rows=rows, classes=_spread(rng, 700, 60000) if rng.random() < 0.5 else VOCAB,
                    k=_spread(rng, 1, 128), temperature=rng.choice([1.0, 1.5, 2.0, 4.0]), padded=rng.random() < 0.5)
        if op == "distil":
            case.update(rest=rng.random() < 0.5, weighted=rng.random() < 0.5)
        return case
    dim = rng.choice([32, 64, 64, 128, 128])
    kv = rng.choice([1, 2, 4, 8, 12])
    group = rng.choice([1, 2, 3, 4, 8]) if kv <= 4 else rng.choice([1, 2, 4])
    case = dict(op=op, dtype=dtype, heads=kv * group, kv_heads=kv, dim=dim)
    kind = rng.choice(["step", "train", "train", "prompt"])
    if kind == "step":               # single tokens or a few at once, against caches
        lo = _spread(rng, 1, 4000)
        seqs, few = _spread(rng, 1, 48), rng.choice([1, 1, 1, 3])
        hi = min(lo * rng.choice([2, 6]) + 4, 160000 // seqs + 4)
        case.update(seqs=seqs, q_min=1, q_max=few, k_min=min(lo, hi), k_max=hi, causal=True, slots=rng.random() < 0.5,
                    train=False)
        return case
    lo = _spread(rng, 1, 1200)
    hi = lo * rng.choice([1, 2, 6]) + rng.choice([0, 5])
    tokens = 12000 if dtype == "bf16" else 3000
    hi = min(hi, tokens // 2)
    seqs = _spread(rng, 1, max(1, min(400, tokens // hi)))
    cross = rng.random() < 0.25
    case.update(seqs=seqs, q_min=min(lo, hi), q_max=hi, k_min=_spread(rng, 1, 300) if cross else 0, k_max=400 if cross else 0,
                causal=False if cross else rng.random() < 0.8, slots=False, train=kind == "train")
    return case


def _lengths(case):
    """(query lengths, key lengths) of the case's sequences"""
    rng = random.Random("%d %d %d %d %d" % tuple(case[n] for n in ("seqs", "q_min", "q_max", "k_min", "k_max")))
    lq = [_spread(rng, case["q_min"], case["q_max"]) for _ in range(case["seqs"])]
    if not case["k_max"]:
        return lq, list(lq)
    lk = [_spread(rng, case["k_min"], case["k_max"]) for _ in range(case["seqs"])]
    return lq, ([max(a, b) for a, b in zip(lq, lk)] if case["causal"] else lk)


def _dtype(case):
    return torch.bfloat16 if case["dtype"] == "bf16" else torch.float32


# ---------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------
def _starts(lengths):
    out = [0]
    for n in lengths:
        out.append(out[-1] + n)
    return out


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *shape: torch.randn(shape, generator=gen, device="cuda")
    dt = _dtype(case)
    state = {"case": case}
    if case["op"] == "attention":
        lq, lk = _lengths(case)
        # slots: every sequence of a cache has the same room, of which its length is filled
        room = [max(lk) + 7] * len(lk) if case["slots"] else lk
        H, G, D = case["heads"], case["kv_heads"], case["dim"]
        nq, nk = sum(lq), sum(room)
        state.update(lq=lq, lk=lk, k_starts=_starts(room)[:-1],
                     cu_q=torch.tensor(_starts(lq), dtype=torch.int32, device="cuda"),
                     cu_k=torch.tensor(_starts(room), dtype=torch.int32, device="cuda"),
                     k_lens=torch.tensor(lk, dtype=torch.int32, device="cuda") if case["slots"] else None)
        if not case["k_max"]:            # one projection's output: q | k | v side by side in a row
            qkv = (normal(nq, H + 2 * G, D) * 1.2).to(dt)
            q, k, v = qkv[:, :H], qkv[:, H:H + G], qkv[:, H + G:]
        else:
            q, k, v = ((normal(n, h, D) * 1.2).to(dt) for n, h in ((nq, H), (nk, G), (nk, G)))
        if case["train"]:
            state["dout"] = normal(nq, H, D).to(dt)
            q, k, v = (t.detach().requires_grad_() for t in (q, k, v))
        state.update(q=q, k=k, v=v)
        return state
    R, N, K = case["rows"], case["classes"], case["k"]
    width = (N + 7) // 8 * 8 if case["padded"] else N

    def rows(x):
        buf = torch.zeros((R, width), dtype=dt, device="cuda")
        buf[:, :N] = x.to(dt)
        return buf[:, :N]
    # a few likely classes over a broad floor
    base = normal(R, N) * 1.8
    hot = torch.randint(0, N, (R, 12), generator=gen, device="cuda")
    base.scatter_add_(1, hot, 5.0 * torch.rand((R, 12), generator=gen, device="cuda") + 3.0)
    if case["op"] == "top":
        state["logits"] = rows(base)
        return state
    student = rows(base * 0.8 + 0.9 * normal(R, N))
    values, classes = torch.topk(base.to(dt).float(), K, dim=1)
    state.update(student=student.detach().requires_grad_(), values=values.contiguous(), classes=classes.to(torch.int32),
                 lse=torch.logsumexp(base.to(dt).float() / case["temperature"], dim=1) if case["rest"] else None,
                 weight=torch.rand(R, generator=gen, device="cuda") + 0.1 if case["weighted"] else None)
    return state


# ---------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------
def run(state):
    case = state["case"]
    if own:
        return _run_own(case, state)
    with torch.no_grad():
        return {"attention": _plain_attention, "top": _plain_top, "distil": _plain_distil}[case["op"]](case, state)


def _run_own(case, st):
    from efficientvlm_amd import ops
    if case["op"] == "attention":
        args = (st["q"], st["k"], st["v"], st["cu_q"], st["cu_k"])
        if not case["train"]:
            with torch.no_grad():
                return (ops.packed_attention(*args, k_lens=st["k_lens"], causal=case["causal"]),)
        out = ops.packed_attention(*args, k_lens=st["k_lens"], causal=case["causal"])
        return (out.detach(),) + torch.autograd.grad(out, args[:3], st["dout"])
    if case["op"] == "top":
        return ops.top_logits(st["logits"], case["k"], temperature=case["temperature"])
    loss = ops.soft_cross_entropy_top(st["student"], st["values"], st["classes"], lse=st["lse"],
                                      temperature=case["temperature"], row_weight=st["weight"])
    return (loss.detach(),) + torch.autograd.grad(loss, (st["student"],))


def _plain_attention(case, st):
    lq, lk = st["lq"], st["lk"]
    S, H, G, D = len(lq), case["heads"], case["kv_heads"], case["dim"]
    q, k, v, dout = st["q"], st["k"], st["v"], st.get("dout")
    q0, k0 = _starts(lq), st["k_starts"]
    out = torch.zeros_like(q, memory_format=torch.contiguous_format)
    grads = [torch.zeros_like(t, memory_format=torch.contiguous_format) for t in (q, k, v)] if case["train"] else []
    # many short sequences go through one padded batch, long ones one by one
    together = S if S * H * max(lq) * max(lk) <= 1 << 27 else 1
    for s in range(0, S, together):
        part = slice(s, s + together)
        mq, mk = max(lq[part]), max(lk[part])
        iq = torch.arange(mq, device="cuda")
        ik = torch.arange(mk, device="cuda")
        nq = torch.tensor(lq[part], device="cuda")[:, None]
        nk = torch.tensor(lk[part], device="cuda")[:, None]
        in_q, in_k = iq < nq, ik < nk
        at_q = (torch.tensor(q0[s:s + together], device="cuda")[:, None] + iq).where(in_q, 0)
        at_k = (torch.tensor(k0[part], device="cuda")[:, None] + ik).where(in_k, 0)
        seen = in_k[:, None, :] & in_q[:, :, None]
        if case["causal"]:
            seen = seen & (ik[None, None, :] <= iq[None, :, None] + (nk - nq)[:, :, None])
        seen = seen[:, None, None]
        # [sequence, key head, heads that share it, token, D]
        Q = q[at_q].float().unflatten(2, (G, H // G)).permute(0, 2, 3, 1, 4)
        K = k[at_k].float().permute(0, 2, 1, 3)[:, :, None]
        V = v[at_k].float().permute(0, 2, 1, 3)[:, :, None]
        scale = D ** -0.5
        P = (torch.matmul(Q, K.transpose(-1, -2)) * scale).masked_fill(~seen, float("-inf"))
        P = (P - P.amax(-1, keepdim=True).clamp_min(-1e30)).exp()
        P = P / P.sum(-1, keepdim=True).clamp_min(1e-30)
        O = torch.matmul(P, V)
        back = lambda x, inside: x.flatten(2, 3)[inside] if x.dim() == 5 else x[inside]
        out[at_q[in_q]] = back(O.permute(0, 3, 1, 2, 4), in_q).to(q.dtype)
        if not case["train"]:
            continue
        dO = dout[at_q].float().unflatten(2, (G, H // G)).permute(0, 2, 3, 1, 4)
        dP = torch.matmul(dO, V.transpose(-1, -2))
        dV = torch.matmul(P.transpose(-1, -2), dO * in_q[:, None, None, :, None]).sum(2)
        dS = P * (dP - (dO * O).sum(-1, keepdim=True)) * scale
        dQ = torch.matmul(dS, K)
        dK = torch.matmul(dS.transpose(-1, -2), Q).sum(2)
        grads[0][at_q[in_q]] = back(dQ.permute(0, 3, 1, 2, 4), in_q).to(q.dtype)
        grads[1][at_k[in_k]] = back(dK.permute(0, 2, 1, 3), in_k).to(q.dtype)
        grads[2][at_k[in_k]] = back(dV.permute(0, 2, 1, 3), in_k).to(q.dtype)
    return (out,) + tuple(grads)


def _plain_top(case, st):
    x = st["logits"].float()
    N = x.shape[1]
    # order of the values as whole numbers, the lower class first among equal values
    bits = (x + 0.0).view(torch.int32)
    key = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long() * (1 << 20) + (N - 1 - torch.arange(N, device="cuda"))
    classes = torch.topk(key, case["k"], dim=1).indices
    y = x * (1.0 / case["temperature"])
    top = y.amax(1, keepdim=True)
    lse = (y - top).exp().sum(1).log() + top[:, 0]
    return x.gather(1, classes), classes.to(torch.int32), lse


def _plain_distil(case, st):
    mul = 1.0 / case["temperature"]
    x = st["student"]
    R, N = x.shape
    y = x.float() * mul
    top = y.amax(1, keepdim=True)
    e = (y - top).exp()
    lse = e.sum(1, keepdim=True).log() + top
    at = st["classes"].long()
    z = st["values"] * mul
    logq = y.gather(1, at) - lse
    if case["rest"]:
        logp = z - st["lse"][:, None]
    else:
        high = z.amax(1, keepdim=True)
        logp = z - (z - high).exp().sum(1, keepdim=True).log() - high
    p = logp.exp()
    row = (p * (logp - logq)).sum(1)
    grad = (y - lse).exp()
    if case["rest"]:
        rest = y.scatter(1, at, float("-inf"))
        lse_rest = (rest - top).exp().sum(1, keepdim=True).log() + top
        p_rest = -torch.expm1(torch.logsumexp(logp, 1, keepdim=True)).clamp_max(0.0)
        row = row + (p_rest * (p_rest.clamp_min(1e-38).log() - (lse_rest - lse)))[:, 0]
        grad = grad - p_rest * (rest - lse_rest).exp()
    grad.scatter_add_(1, at, -p)
    w = st["weight"] if st["weight"] is not None else torch.ones(R, device="cuda")
    return (row * w).sum() / R, (grad * (w * (mul / R))[:, None]).to(x.dtype)


# ---------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------------
def work(case):
    size = 2 if case["dtype"] == "bf16" else 4
    if case["op"] != "attention":
        cells, kept = case["rows"] * case["classes"], case["rows"] * case["k"]
        if case["op"] == "top":
            return {"bytes": cells * size + kept * 8 + case["rows"] * 4, "flops": 4 * cells}
        extra = case["rows"] * 4 * (int(case["rest"]) + int(case["weighted"]))
        return {"bytes": 2 * cells * size + kept * 8 + extra, "flops": 8 * cells}
    lq, lk = _lengths(case)
    H, G, D = case["heads"], case["kv_heads"], case["dim"]
    if case["causal"]:                    # query i of a sequence sees lk - lq + i + 1 keys
        pairs = sum(a * (b - a) + a * (a + 1) // 2 for a, b in zip(lq, lk))
    else:
        pairs = sum(a * b for a, b in zip(lq, lk))
    q_bytes, k_bytes = sum(lq) * H * D * size, sum(lk) * G * D * size
    if case["train"]:                     # q, k, v, dO in; O, dQ, dK, dV out; two products forward, five backward
        return {"bytes": 4 * q_bytes + 4 * k_bytes, "flops": 14 * pairs * H * D}
    return {"bytes": 2 * q_bytes + 2 * k_bytes, "flops": 4 * pairs * H * D}


# ---------------------------------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------------------------------
def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "top":
        x = st["logits"].double()
        order = torch.sort(x, dim=1, descending=True, stable=True)
        return (order.values[:, :case["k"]], order.indices[:, :case["k"]].to(torch.int32),
                torch.logsumexp(x / case["temperature"], 1))
    if case["op"] == "distil":
        return _exact_distil(case, st)
    lq, lk = st["lq"], st["lk"]
    share = case["heads"] // case["kv_heads"]
    q, k, v = (st[n].detach() for n in "qkv")
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    dq, dk, dv = (torch.zeros(t.shape, dtype=torch.float64, device="cuda") for t in (q, k, v))
    a = 0
    for s, (n, m) in enumerate(zip(lq, lk)):
        b = st["k_starts"][s]
        hidden = None
        if case["causal"]:
            hidden = torch.ones((n, m), dtype=torch.bool, device="cuda").triu_(m - n + 1)
        # as many key heads at once as fit into 4 GB of scores
        step = max(1, min(case["kv_heads"], (1 << 29) // (n * m * share)))
        for h in range(0, case["kv_heads"], step):
            g = min(step, case["kv_heads"] - h)
            heads = slice(h * share, (h + g) * share)
            Q = q[a:a + n, heads].double().transpose(0, 1).reshape(g, share * n, -1)
            K = k[b:b + m, h:h + g].double().transpose(0, 1).contiguous()
            V = v[b:b + m, h:h + g].double().transpose(0, 1).contiguous()
            scores = torch.bmm(Q, K.transpose(1, 2).contiguous()) / math.sqrt(case["dim"])
            if hidden is not None:
                scores.view(g, share, n, m).masked_fill_(hidden, -math.inf)
            probs = torch.softmax(scores, dim=2)
            del scores
            ctx = torch.bmm(probs, V)
            out[a:a + n, heads] = ctx.view(g * share, n, -1).transpose(0, 1)
            if case["train"]:
                dctx = st["dout"][a:a + n, heads].double().transpose(0, 1).reshape(g, share * n, -1)
                dv[b:b + m, h:h + g] = torch.bmm(probs.transpose(1, 2).contiguous(), dctx).transpose(0, 1)
                dprobs = torch.bmm(dctx, V.transpose(1, 2).contiguous())
                dscores = probs * (dprobs - (dprobs * probs).sum(2, keepdim=True)) / math.sqrt(case["dim"])
                del dprobs
                dq[a:a + n, heads] = torch.bmm(dscores, K).view(g * share, n, -1).transpose(0, 1)
                dk[b:b + m, h:h + g] = torch.bmm(dscores.transpose(1, 2).contiguous(), Q).transpose(0, 1)
        a += n
    return (out, dq, dk, dv) if case["train"] else (out,)


def _exact_distil(case, st):
    T = case["temperature"]
    R, N = st["student"].shape
    w = st["weight"].double() if st["weight"] is not None else torch.ones(R, dtype=torch.float64, device="cuda")
    loss, grads = 0.0, []
    for r in range(0, R, 512):
        part = slice(r, r + 512)
        x = st["student"][part].detach().double().requires_grad_()
        at = st["classes"][part].long()
        teacher = st["values"][part].double() / T
        logq = torch.log_softmax(x / T, 1)
        kept = logq.gather(1, at)
        if case["rest"]:
            logp = teacher - st["lse"][part].double()[:, None]
            other = torch.ones_like(logq, dtype=torch.bool).scatter_(1, at, False)
            q_rest = torch.logsumexp(logq.masked_fill(~other, -math.inf), 1)
            p_rest = (1.0 - logp.exp().sum(1)).clamp_min(0.0)
            last = torch.xlogy(p_rest, p_rest) - p_rest * q_rest
        else:
            logp = torch.log_softmax(teacher, 1)
            last = 0.0
        total = ((logp.exp() * (logp - kept)).sum(1) + last).mul(w[part]).sum() / R
        grads.append(torch.autograd.grad(total, x)[0])
        loss = loss + total.detach()
    return loss, torch.cat(grads)
