"""ops.packed_attention against its definition in 64 bits.

Tolerances count roundings (u = half a step of the storage type: 2^-8 bf16, 2^-24 f32) and are per element:
  probability p_ij        relative error rel_i: the scores' f32 dot products ((dh + 8) 2^-24 scale sum_d |q_d k_d|, twice: for the score
                          and for the maximum / log-sum-exp), the f32 sums over n keys and the 2^x / division ((n + 16) 2^-24);
                          rounded once more to the storage type as an operand of the next product (u)
  O                       u |O| + (u + rel_i) sum_j p |v|
  delta = dO.O            with the stored O: sum_d |dO| (error of O) + dh 2^-24 sum_d |dO O|            =: e_i
  dS = p (dP - delta)     u |dS| + rel_i p (|dP| + |delta|) + p (e_i + (dh + 8) 2^-24 sum_d |dO v|)     =: f_ij
  dQ, dK, dV              u |x| + sum of the operands' errors, + (n + 16) 2^-24 of the absolute sum (n terms summed in f32)
"""
import ctypes
import math
import os
import re

import pytest
import torch

from efficientvlm_amd import ops

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BF16, F32 = torch.bfloat16, torch.float32
F = 2.0 ** -24


def starts(lens, first=0):
    out = [first]
    for n in lens:
        out.append(out[-1] + n)
    return out


def definition(q, k, v, dout, q0, lq, k0, lk, causal, scale, u):
    """(O, dQ, dK, dV) in 64 bits and the bound of each element's error, on the CPU"""
    q, k, v = (t.detach().double().cpu() for t in (q, k, v))
    dout = torch.zeros_like(q) if dout is None else dout.detach().double().cpu()
    H, dh = q.shape[1:]
    G = H // k.shape[1]
    val = [torch.zeros_like(t) for t in (q, q, k, v)]
    tol = [torch.zeros_like(t) for t in (q, q, k, v)]
    for a, n, b, m in zip(q0, lq, k0, lk):
        if n == 0 or m == 0:
            continue
        seen = torch.ones(n, m, dtype=torch.bool)
        if causal:
            seen = torch.arange(m)[None, :] <= torch.arange(n)[:, None] + (m - n)
        for h in range(H):
            Q, dO = q[a:a + n, h], dout[a:a + n, h]
            K, V = k[b:b + m, h // G], v[b:b + m, h // G]
            S = (Q @ K.T * scale).masked_fill(~seen, -math.inf)
            P = torch.softmax(S, 1).nan_to_num(0.0)                  # (rows that see nothing)
            O = P @ V
            rel = (2 * (dh + 8) * F * scale * (Q.abs() @ K.abs().T)).masked_fill(~seen, 0).amax(1) + (m + 16) * F
            A = P @ V.abs()
            eO = u * O.abs() + (u + rel)[:, None] * A
            dP = dO @ V.T
            delta = (dO * O).sum(1)
            dS = P * (dP - delta[:, None])
            e = (dO.abs() * eO).sum(1) + dh * F * (dO * O).abs().sum(1)
            f = (u * dS.abs() + rel[:, None] * P * (dP.abs() + delta.abs()[:, None])
                 + P * (e[:, None] + (dh + 8) * F * (dO.abs() @ V.abs().T)))
            absS = P * (dP.abs() + delta.abs()[:, None])
            val[0][a:a + n, h], tol[0][a:a + n, h] = O, eO
            x = scale * dS @ K
            val[1][a:a + n, h], tol[1][a:a + n, h] = x, u * x.abs() + scale * ((f + (m + 16) * F * absS) @ K.abs())
            rows = G * n + 16
            val[2][b:b + m, h // G] += scale * dS.T @ Q
            tol[2][b:b + m, h // G] += scale * (f + rows * F * absS).T @ Q.abs()
            val[3][b:b + m, h // G] += P.T @ dO
            tol[3][b:b + m, h // G] += ((u + rel[:, None] + rows * F) * P).T @ dO.abs()
    tol[2] += u * val[2].abs()
    tol[3] += u * val[3].abs()
    return val, tol


def check(got, val, tol, names=("O", "dQ", "dK", "dV")):
    for g, x, t, n in zip(got, val, tol, names):
        g = g.detach().double().cpu()
        assert g.shape == x.shape
        over = ((g - x).abs() - t - 1e-30).nan_to_num(math.inf)
        assert over.max() <= 0, f"{n}: {int((over > 0).sum())} of {over.numel()} elements off, worst by {over.max():.3e} over its bound"


def problem(dtype, H, Hkv, dh, lq, lk=None, slots=0, before=0, behind=0, seed=0, layout="plain"):
    """q, k, v, dout, the starts and lengths; `slots`: room behind every key range, `before` / `behind`: rows outside"""
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)
    same = lk is None
    lk = list(lq) if same else list(lk)
    room = [n + slots for n in lk]
    q0, k0 = starts(lq, before), starts(room, before if same and not slots else 0)
    nq = q0[-1] + behind
    nk = nq if same and not slots else k0[-1] + behind
    if layout == "qkv" and nq == nk:
        buf = r(nq, H + 2 * Hkv, dh).to(dtype).cuda()
        q, k, v = buf[:, :H], buf[:, H:H + Hkv], buf[:, H + Hkv:]
    elif layout == "heads_first":                 # [heads, tokens, dh] storage
        q, k, v = (r(h, n, dh).to(dtype).cuda().transpose(0, 1) for h, n in ((H, nq), (Hkv, nk), (Hkv, nk)))
    elif layout == "odd":                         # rows that are no whole 16-byte pieces: copied by the call
        q, k, v = (r(n, h, dh + 1).to(dtype).cuda()[..., 1:] for h, n in ((H, nq), (Hkv, nk), (Hkv, nk)))
    else:
        q, k, v = (r(n, h, dh).to(dtype).cuda() for h, n in ((H, nq), (Hkv, nk), (Hkv, nk)))
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    return dict(q=q, k=k, v=v, dout=r(nq, H, dh).to(dtype).cuda(), cu_q=i32(q0), cu_k=i32(k0),
                k_lens=i32(lk) if slots else None, q0=q0[:-1], lq=list(lq), k0=k0[:-1], lk=lk)


def run(p, causal=True, scale=None, backward=True):
    q, k, v = (p[n].detach().requires_grad_(backward) for n in "qkv")
    out = ops.packed_attention(q, k, v, p["cu_q"], p["cu_k"], k_lens=p["k_lens"], scale=scale, causal=causal)
    return (out,) + (torch.autograd.grad(out, (q, k, v), p["dout"]) if backward else ())


def both(p, causal=True, scale=None, backward=True):
    u = 2.0 ** -8 if p["q"].dtype == BF16 else F
    sc = p["q"].shape[2] ** -0.5 if scale is None else scale
    val, tol = definition(p["q"], p["k"], p["v"], p["dout"] if backward else None, p["q0"], p["lq"], p["k0"], p["lk"], causal, sc, u)
    got = run(p, causal, scale, backward)
    check(got, val, tol)
    return got, val, tol


# ---- refusals (no GPU) ------------------------------------------------------------------------------
def test_refusals():
    t = lambda *s, dt=F32: torch.zeros(*s, dtype=dt)
    cu = torch.tensor([0, 4], dtype=torch.int32)
    ok = dict(q=t(4, 4, 16), k=t(4, 2, 16), v=t(4, 2, 16), cu_q=cu)
    with pytest.raises(RuntimeError, match="GPU only"):
        ops.packed_attention(**ok)
    bad = [(dict(q=t(4, 64)), RuntimeError, "tokens, heads"), (dict(k=t(4, 3, 16), v=t(4, 3, 16)), RuntimeError, "multiple"),
           (dict(v=t(4, 2, 16, dt=BF16)), TypeError, "one dtype"), (dict(v=t(5, 2, 16)), RuntimeError, "agree"),
           (dict(q=t(4, 4, 24)), RuntimeError, "head dim 24"), (dict(k=t(5, 2, 16), v=t(5, 2, 16)), RuntimeError, "as many keys"),
           (dict(cu_q=cu.long()), TypeError, "int32"), (dict(cu_k=torch.zeros(3, dtype=torch.int32)), RuntimeError, "entries"),
           (dict(k_lens=torch.zeros(2, dtype=torch.int32)), RuntimeError, "entries"), (dict(cu_q=cu[:0]), RuntimeError, "entries"),
           (dict(scale=0.0), RuntimeError, "scale"), (dict(scale=-1.0), RuntimeError, "scale"), (dict(scale=math.nan), RuntimeError, "scale")]
    for change, err, match in bad:
        with pytest.raises(err, match=match):
            ops.packed_attention(**{**ok, **change})
    for d in (12, 136):
        with pytest.raises(RuntimeError, match="head dim"):
            ops.packed_attention(t(4, 4, d), t(4, 2, d), t(4, 2, d), cu)
    with pytest.raises(TypeError, match="float16"):
        ops.packed_attention(*(t(4, 2, 16, dt=torch.float16) for _ in range(3)), cu)


def test_c_entry_refuses_before_any_launch():
    """the C entries check what a kernel assumes on the host; nothing reaches a device here"""
    from efficientvlm_amd import _lib
    lib = _lib.load()
    base = dict(dtype=_lib.BF16, Tq=4, Tk=4, S=1, H=4, Hkv=2, dh=64, scale=0.125, Q=4096, K=4096, V=4096, O=4096, cu_q=4096, cu_k=4096,
                q_tok=256, q_head=64, k_tok=128, k_head=64, v_tok=128, v_head=64)
    for change in (dict(dtype=7), dict(dh=72 + 4), dict(dh=136), dict(H=5), dict(scale=0.0), dict(Q=4098), dict(k_tok=12), dict(O=None),
                   dict(cu_q=None), dict(K=None), dict(Tq=-1)):
        a = _lib.PackedAttnArgs(**{**base, **change})
        assert lib.evlm_packed_attention_fwd(ctypes.byref(a), None) != 0, change
        assert lib.evlm_last_error()
    assert lib.evlm_packed_attention_bwd(ctypes.byref(_lib.PackedAttnArgs(**base)), None) != 0       # no dO, lse, ...
    assert lib.evlm_packed_attention_fwd(ctypes.byref(_lib.PackedAttnArgs(**{**base, "Tq": 0})), None) == 0


def test_struct_layout_matches_header():
    from efficientvlm_amd import _lib
    src = open(os.path.join(ROOT, "include", "evlm_hip.h")).read()
    body = re.search(r"typedef struct \{((?:(?!typedef struct).)*?)\}\s*evlm_packed_attn_args", src, flags=re.S).group(1)
    fields = []
    for decl in re.sub(r"/\*.*?\*/", "", body, flags=re.S).split(";"):
        names = re.sub(r"^(const\s+)?[A-Za-z_0-9]+\s*\**", "", decl.strip())
        fields += [n.strip().lstrip("*").strip() for n in re.sub(r"(const\s+)?\bvoid\*|int32_t\*", "", names).split(",") if n.strip()]
    assert fields == [f[0] for f in _lib.PackedAttnArgs._fields_]


# ---- values and gradients ---------------------------------------------------------------------------
LENGTHS = {
    "ones": [1] * 9,
    "answers": [3, 7, 1, 12, 5, 0, 16, 2, 9, 4],
    "edges": [31, 32, 33, 0, 1, 127, 128, 129, 63, 65],
    "one_long": [517],
    "ragged": [200, 3, 90, 1, 333],
}


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lengths", sorted(LENGTHS))
def test_lengths(dtype, causal, lengths):
    both(problem(dtype, 4, 2, 64, LENGTHS[lengths]), causal)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("heads", [(1, 1), (3, 1), (12, 12), (10, 2), (14, 2), (32, 1), (40, 1), (71, 1)])
def test_head_groups(dtype, heads):
    both(problem(dtype, heads[0], heads[1], 32, [17, 40, 1, 70], seed=heads[0]))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("dh", [8, 24, 40, 64, 72, 96, 128])
def test_head_dims(dtype, dh):
    both(problem(dtype, 4, 2, dh, [50, 1, 140], seed=dh))
    both(problem(dtype, 4, 2, dh, [5, 1, 9, 2], seed=dh))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("causal", [True, False])
def test_other_keys_and_rows_that_see_none(dtype, causal):
    """more keys than queries (a chunk behind a cache), fewer (causal: the first queries see nothing), none at all"""
    (out, dq, dk, dv), _, _ = both(problem(dtype, 6, 2, 64, [4, 20, 9, 1, 0, 70, 3], [40, 5, 0, 300, 7, 70, 1]), causal)
    if causal:
        assert (out[4:4 + 15] == 0).all() and (dq[4:4 + 15] == 0).all()           # 20 queries, 5 keys
    assert (out[24:33] == 0).all() and (dq[24:33] == 0).all()                     # no keys
    assert (dk[345:352] == 0).all() and (dv[345:352] == 0).all()                  # no queries


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("heads,dh", [((12, 12), 64), ((32, 8), 128), ((8, 1), 128), ((6, 2), 40)])
@pytest.mark.parametrize("lk", [[1, 2, 31], [33, 64, 500, 0, 1], [9000, 4097], [20000]])
def test_single_tokens_behind_caches(dtype, heads, dh, lk):
    both(problem(dtype, *heads, dh, [1] * len(lk), lk, slots=9), backward=False)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_few_tokens_behind_caches_train(dtype):
    both(problem(dtype, 8, 2, 64, [1, 3, 2], [1500, 700, 2100], slots=5))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("heads,dh,lq,lk", [
    ((2, 1), 128, [255, 256, 257, 31, 1], None),                         # blocks of 256 keys and of 128
    ((4, 1), 128, [600, 90], None),                                      # ... their rows shared by several blocks
    ((4, 1), 128, [20, 47, 1, 33], None),                                # ... and of 32
    ((2, 2), 64, [150, 161, 32, 33], None),                              # one wave a block of keys, several blocks
    ((2, 2), 64, [300, 210, 128], None),                                 # four waves a block of keys
    ((4, 2), 64, [3, 1, 0, 30, 17], [65, 700, 100, 333, 0]),             # few queries: keys split over the waves
    ((4, 2), 128, [3, 1, 0, 30, 17], [65, 700, 100, 333, 0]),
    ((8, 8), 32, [7] * 135, [70] * 134 + [40]),                          # ... enough blocks without; sequences counted four a lane
    ((2, 1), 64, [9, 40, 1] * 30, None),                                 # 90 sequences, in order
])
def test_forms_of_the_work(dtype, causal, heads, dh, lq, lk):
    """lengths around the sizes at which the kernels cut the work differently"""
    both(problem(dtype, *heads, dh, lq, lk, seed=len(lq)), causal)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("parts", [1, 3, 4, 7, 8, 9, 30, 75])
def test_chunks_of_keys_joined(dtype, parts):
    """a single token over so many chunks (one chunk a head group is at least 256 keys)"""
    both(problem(dtype, 2, 1, 72, [1, 2], [256 * parts, 600], slots=3), backward=False)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("layout", ["qkv", "heads_first", "odd"])
def test_layouts(dtype, layout):
    p = problem(dtype, 4, 2, 64, [40, 9, 150], layout=layout)
    p["dout"] = p["dout"].transpose(0, 1).contiguous().transpose(0, 1)
    both(p)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("lq", [[5, 3], [150, 40]])
def test_rows_outside_all_sequences(dtype, lq):
    """rows before the first and behind the last sequence: zero outputs and gradients, whatever they hold"""
    p = problem(dtype, 4, 2, 64, lq, before=3, behind=37)
    inside = torch.zeros(p["q"].shape[0], dtype=torch.bool, device="cuda")
    inside[3:3 + sum(lq)] = True
    for n in "qkv":
        p[n][~inside] = math.nan
    p["dout"][~inside] = math.nan
    got = run(p)
    for t in got:
        assert (t[~inside] == 0).all()
    q = dict(p)
    for n in ("q", "k", "v", "dout"):
        q[n] = p[n].masked_fill(~inside[:, None, None], 0.0)
    for a, b in zip(got, run(q)):
        assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("lq,lk", [([1, 1, 1], [40, 3, 2000]), ([60, 5, 130], [70, 5, 333])])
def test_unfilled_room_and_neighbours_are_not_read(dtype, lq, lk):
    """NaN behind the filled part of the slots, and NaN in ONE sequence, stay where they are"""
    p = problem(dtype, 4, 2, 64, lq, lk, slots=11)
    want = run(p)
    for b, n in zip(p["k0"], p["lk"]):
        for t in ("k", "v"):
            p[t][b + n:b + n + 11] = math.nan
    got = run(p)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    assert all((got[i][b + n:b + n + 11] == 0).all() for i in (2, 3) for b, n in zip(p["k0"], p["lk"]))
    p["v"][p["k0"][1]] = math.nan                                                # a key every row of sequence 1 sees
    got = run(p)
    a, n = p["q0"][1], p["lq"][1]
    assert got[0][a:a + n].isnan().all()
    keep = torch.ones(got[0].shape[0], dtype=torch.bool, device="cuda")
    keep[a:a + n] = False
    assert torch.equal(got[0][keep], want[0][keep]) and torch.equal(got[1][keep], want[1][keep])


@pytest.mark.gpu
def test_scores_far_apart_and_infinite():
    """scores whose differences pass 2^100, and keys with -inf scores: an exact 0, no NaN"""
    p = problem(F32, 2, 2, 64, [70], seed=3)
    p["q"] = p["q"].abs()
    p["k"] = p["k"] * 40
    both(p, scale=1.0)
    p = problem(F32, 2, 1, 64, [1, 40], [50, 90], seed=4)
    p["q"] = p["q"].abs() + 0.1
    low = [3, 60, 61]
    want = {n: p[n].clone() for n in "kv"}
    for j in low:
        p["k"][j] = -math.inf
    got = run(p, causal=False, backward=False)[0]
    assert got.isfinite().all()
    S = (p["q"].double().cpu().transpose(0, 1) @ p["k"].double().cpu()[:, 0].T.nan_to_num(neginf=-1e300)) / 8
    ref = []
    for i in range(41):
        b, n = (0, 50) if i == 0 else (50, 90)
        ref.append(torch.softmax(S[:, i, b:b + n], 1) @ want["v"].double().cpu()[b:b + n, 0])
    err = (got.double().cpu() - torch.stack(ref)).abs().max()
    assert err <= 200 * F * want["v"].abs().max().item() * 8             # (n + dh + scores' size) roundings of values up to max |v|


@pytest.mark.gpu
def test_gradient_against_differences():
    """directional differences of the definition in 64 bits (step 1e-5: truncation ~ 1e-10) against the f32 kernels' gradients"""
    p = problem(F32, 4, 2, 32, [30, 1, 45, 7], seed=5)
    got = run(p)
    val, tol = definition(p["q"], p["k"], p["v"], p["dout"], p["q0"], p["lq"], p["k0"], p["lk"], True, 32 ** -0.5, F)

    def loss(**move):
        x = {n: p[n].double() + (1e-5 * move[n] if n in move else 0) for n in "qkv"}
        o = definition(x["q"], x["k"], x["v"], None, p["q0"], p["lq"], p["k0"], p["lk"], True, 32 ** -0.5, F)[0][0]
        return (o * p["dout"].double().cpu()).sum()
    for i, n in enumerate("qkv"):
        d = torch.randn(p[n].shape, generator=torch.Generator().manual_seed(i), dtype=torch.float64)
        diff = (loss(**{n: d.cuda()}) - loss(**{n: -d.cuda()})) / 2e-5
        mine = (got[1 + i].double().cpu() * d).sum()
        assert abs(mine - diff) <= (tol[1 + i] * d.abs()).sum() + 1e-7 * (1 + abs(diff))


# ---- how it is called -------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("lq", [[4, 9, 2], [300, 130]])
def test_same_bits_every_time(lq):
    p = problem(BF16, 8, 2, 64, lq)
    first = run(p)
    for _ in range(3):
        for a, b in zip(run(p), first):
            assert torch.equal(a, b)


@pytest.mark.gpu
def test_only_some_gradients_and_no_grad():
    p = problem(BF16, 4, 2, 64, [30, 80])
    want = run(p)
    k = p["k"].detach().requires_grad_()
    out = ops.packed_attention(p["q"], k, p["v"], p["cu_q"])
    assert torch.equal(out, want[0])
    out.backward(p["dout"])
    assert torch.equal(k.grad, want[2])
    with torch.no_grad():
        out = ops.packed_attention(p["q"], k, p["v"], p["cu_q"])
    assert not out.requires_grad and torch.equal(out, want[0])
    with pytest.raises(RuntimeError, match="second derivative"):
        q = p["q"].float().detach().requires_grad_()
        g, = torch.autograd.grad(ops.packed_attention(q, p["k"].float(), p["v"].float(), p["cu_q"]).sum(), q, create_graph=True)
        g.sum().backward()


@pytest.mark.gpu
def test_gradients_of_shared_storage_and_broadcast():
    """slices of one projection and key heads broadcast from one: autograd sums what the call hands back"""
    p = problem(F32, 4, 4, 32, [20, 33])
    one = p["k"][:, :1].contiguous().detach().requires_grad_()
    out = ops.packed_attention(p["q"], one.expand(-1, 4, -1), p["v"], p["cu_q"])
    out.backward(p["dout"])
    full = p["k"][:, :1].expand(-1, 4, -1).contiguous()
    val, tol = definition(p["q"], full, p["v"], p["dout"], p["q0"], p["lq"], p["k0"], p["lk"], True, 32 ** -0.5, F)
    check([one.grad], [val[2].sum(1, keepdim=True)], [tol[2].sum(1, keepdim=True) + 8 * F * val[2].abs().sum(1, keepdim=True)], ["dK"])
    qkv = torch.randn(53, 12, 32, generator=torch.Generator().manual_seed(1)).cuda().requires_grad_()
    ops.packed_attention(qkv[:, :4], qkv[:, 4:8], qkv[:, 8:], p["cu_q"]).sum().backward()       # (dO: an expanded scalar)
    val, tol = definition(qkv[:, :4], qkv[:, 4:8], qkv[:, 8:], torch.ones(53, 4, 32), p["q0"], p["lq"], p["k0"], p["lk"], True, 32 ** -0.5, F)
    check([qkv.grad], [torch.cat(val[1:], 1)], [torch.cat(tol[1:], 1)], ["dQKV"])


@pytest.mark.gpu
def test_nothing_to_do():
    z = lambda *s: torch.zeros(*s, dtype=BF16, device="cuda")
    i = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")
    assert ops.packed_attention(z(0, 4, 64), z(0, 2, 64), z(0, 2, 64), i(0)).shape == (0, 4, 64)
    assert (ops.packed_attention(z(5, 4, 64) + 1, z(5, 2, 64), z(5, 2, 64) + 1, i(0)) == 0).all()             # no sequences
    assert (ops.packed_attention(z(5, 4, 64) + 1, z(0, 2, 64), z(0, 2, 64), i(0, 5), i(0, 0)) == 0).all()     # no keys
    q, k, v = (t.requires_grad_() for t in (z(5, 4, 64), z(7, 2, 64), z(7, 2, 64)))
    out = ops.packed_attention(q, k, v, i(0, 0, 0), i(0, 3, 3))
    out.sum().backward()
    assert all((t == 0).all() for t in (out, q.grad, k.grad, v.grad))
    q, k, v = (t.requires_grad_() for t in (z(0, 4, 64), z(7, 2, 64), z(7, 2, 64)))
    ops.packed_attention(q, k, v, i(0, 0), i(0, 7)).sum().backward()
    assert q.grad.shape == (0, 4, 64) and (k.grad == 0).all() and (v.grad == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("cu_q,cu_k,k_lens", [([0, 99, 20], None, None), ([-5, 30, 12], None, None), ([40, 2, 1], None, None),
                                              ([0, 10, 20], [0, 1 << 30, -7], None), ([0, 10, 20], [0, 10, 20], [1 << 30, -3]),
                                              ([2147483647, -2147483648, 2147483647], None, None)])
def test_starts_that_make_no_sense_stay_inside_the_tensors(cu_q, cu_k, k_lens):
    """clamped on the device: the values are nobody's business, the accesses are"""
    i32 = lambda x: None if x is None else torch.tensor(x, dtype=torch.int32, device="cuda")
    guard = torch.zeros(3, 20, 4, 64, dtype=F32, device="cuda")
    q, k, v = (guard[j].clone().requires_grad_() for j in range(3))
    out = ops.packed_attention(q, k, v, i32(cu_q), i32(cu_k), k_lens=i32(k_lens))
    torch.autograd.grad(out, (q, k, v), torch.ones_like(out))
    torch.cuda.synchronize()
    assert out.shape == (20, 4, 64)


@pytest.mark.gpu
def test_many_sequences():
    """more sequences than one wave counts at a time, empty ones among them"""
    g = torch.Generator().manual_seed(0)
    lens = torch.randint(0, 5, (700,), generator=g).tolist()
    both(problem(BF16, 2, 1, 32, lens))
    both(problem(F32, 2, 2, 32, lens, [3 * n for n in lens]))


@pytest.mark.gpu
@pytest.mark.parametrize("lq,lk", [([5, 9, 2], None), ([140, 60, 33], None), ([1, 1, 1], [3000, 1200, 2])])
def test_capture_follows_the_lengths(lq, lk):
    """one captured forward + backward, replayed on other lengths of the same totals, eager work in between"""
    p = problem(BF16, 8, 2, 64, lq, lk, slots=3 if lk else 0)
    q, k, v = (p[n].detach().clone().requires_grad_() for n in "qkv")

    def step():
        out = ops.packed_attention(q, k, v, p["cu_q"], p["cu_k"], k_lens=p["k_lens"])
        return (out,) + torch.autograd.grad(out, (q, k, v), p["dout"])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        static = step()
    n = sum(lq)
    for turn, cut in enumerate([lq, [1, n - 2, 1] if lk is None else [1, 1, 1], lq]):
        p["cu_q"].copy_(torch.tensor(starts(cut), dtype=torch.int32))
        if lk is None:
            p["cu_k"].copy_(p["cu_q"])
        else:
            p["k_lens"].copy_(torch.tensor([max(1, x - 7 * turn) for x in lk], dtype=torch.int32))
        with torch.no_grad():
            q.copy_(torch.randn(q.shape, generator=torch.Generator().manual_seed(turn)))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in static]
        want = run({**p, "q": q, "k": k, "v": v})
        for a, b in zip(got, want):
            assert torch.equal(a, b)


@pytest.mark.gpu
def test_two_streams_at_once():
    """calls in flight on two streams share nothing"""
    ps = [problem(BF16, 8, 2, 64, [1, 1], [4000, 2500], slots=1, seed=s) for s in range(2)]
    want = [run(p) for p in ps]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in ps]
    got = [None, None]
    for _ in range(5):
        for i, (p, s) in enumerate(zip(ps, streams)):
            with torch.cuda.stream(s):
                got[i] = run(p)
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        for a, b in zip(g, w):
            assert torch.equal(a, b)


@pytest.mark.gpu
def test_keys_behind_two_to_the_31():
    """offsets of a long cache: K is 2^31 + elements, the sequence lies behind them"""
    tokens, Hkv, dh = (1 << 31) // (8 * 128) + 600, 8, 128
    k = torch.zeros(tokens, Hkv, dh, dtype=BF16, device="cuda")
    p = problem(BF16, 8, Hkv, dh, [1, 70], [300, 200])
    k[tokens - 500:] = p["k"]
    cu_k = torch.tensor([tokens - 500, tokens - 200, tokens], dtype=torch.int32, device="cuda")
    got = ops.packed_attention(p["q"], k, k, p["cu_q"], cu_k)
    want = ops.packed_attention(p["q"], p["k"], p["k"], p["cu_q"], p["cu_k"])
    # (the split of the keys over blocks follows the tensors' sizes: equal values, not equal bits)
    val, tol = definition(p["q"], p["k"], p["k"], None, p["q0"], p["lq"], p["k0"], p["lk"], True, dh ** -0.5, 2.0 ** -8)
    check([got], val, tol)
    check([want], val, tol)


# ---- broken values, large scores, wide strides -------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("heads,dh", [((8, 2), 64), ((4, 4), 128)])
def test_a_broken_query_shows_however_long_its_cache(dtype, heads, dh):
    """a NaN in one head's query, NaN in every key, or every score -inf: NaN in exactly the rows of those heads, whether the keys are
    one piece (short caches) or joined from several"""
    for lk in ([20, 33, 5], [3000, 1700, 2000]):
        p = problem(dtype, *heads, dh, [1, 2, 1], lk, slots=5)
        G, b, m = heads[0] // heads[1], p["k0"][1], p["lk"][1]
        for kind in ("query", "keys", "far"):
            clean, q, k = p["q"].clone(), p["q"].clone(), p["k"].clone()
            bad = [(t, h) for t in (1, 2) for h in range(G)]
            if kind == "query":
                q[2, 1, 3] = math.nan
                bad = [(2, 1)]
            elif kind == "keys":
                k[b:b + m, 0] = math.nan
            else:
                clean = q = q.abs() + 0.1
                k[b:b + m, 0] = -math.inf
            got = run({**p, "q": q, "k": k})
            broken = torch.zeros(got[0].shape[:2], dtype=torch.bool, device="cuda")
            for t, h in bad:
                broken[t, h] = True
            assert got[0][broken].isnan().all() and got[1][broken].isnan().all(), (kind, lk)
            val, tol = definition(clean, p["k"], p["v"], p["dout"], p["q0"], p["lq"], p["k0"], p["lk"], True, dh ** -0.5,
                                  2.0 ** -8 if dtype == BF16 else F)
            good = ~broken.cpu()
            check([x[~broken] for x in got[:2]], [x[good] for x in val[:2]], [x[good] for x in tol[:2]])


def test_wide_head_strides_of_keys_are_read_in_place():
    """a cache stored [heads, tokens, dh] has heads 2^22 and more elements apart; only the token stride of K and V is limited, and both
    strides of Q and dO"""
    wide = torch.empty_strided((10, 2, 128), (128, 1 << 22, 1), dtype=BF16)
    x, address, token, head = ops._heads3(wide, keys=True)
    assert x is wide and address == wide.data_ptr() and (token, head) == (128, 1 << 22)
    x, address, token, head = ops._heads3(wide)
    assert x.is_contiguous() and address == x.data_ptr() != wide.data_ptr() and (token, head) == (256, 128)
    apart = torch.empty_strided((2, 2, 128), (1 << 22, 128, 1), dtype=BF16)
    for keys in (False, True):
        x, address, token, head = ops._heads3(apart, keys=keys)
        assert x.is_contiguous() and address == x.data_ptr() != apart.data_ptr() and (token, head) == (256, 128)
    one = apart[:1]                                           # (a single token has no stride)
    assert ops._heads3(one)[1] == one.data_ptr()
    odd = torch.empty(10, 2, 129, dtype=BF16)[..., 1:]
    for keys in (False, True):
        assert ops._heads3(odd, keys=keys)[0].is_contiguous()
    many = torch.empty(2, 1 << 15, 129, dtype=BF16)[..., 1:]  # 2^15 heads of 128: a token stride of 2^22 however it is laid out (the
    x, address, token, head = ops._heads3(many)               # entry refuses it); the address is that of the tensor that is kept
    assert address == x.data_ptr() and (token, head) == (1 << 22, 128)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("lq", [[1, 1], [70, 300]])
def test_heads_first_caches_of_any_length(dtype, lq):
    """K and V with heads 2^22 elements apart: the values of packed ones"""
    p = problem(dtype, 8, 2, 128, lq, [900, 1400])
    tokens = (1 << 15) + 64
    far = {}
    for n in "kv":
        store = torch.zeros(2, tokens, 128, dtype=dtype, device="cuda")
        store[:, :2300] = p[n].transpose(0, 1)
        far[n] = store.transpose(0, 1)
    with torch.no_grad():
        out = ops.packed_attention(p["q"], far["k"], far["v"], p["cu_q"], p["cu_k"])
    val, tol = definition(p["q"], p["k"], p["v"], None, p["q0"], p["lq"], p["k0"], p["lk"], True, 128 ** -0.5,
                          2.0 ** -8 if dtype == BF16 else F)
    check([out], val, tol)
    if lq[0] > 1:
        q, k, v = (t.detach().requires_grad_() for t in (p["q"], far["k"], far["v"]))
        out = ops.packed_attention(q, k, v, p["cu_q"], p["cu_k"])
        got = torch.autograd.grad(out, (q, k, v), p["dout"])
        val, tol = definition(p["q"], p["k"], p["v"], p["dout"], p["q0"], p["lq"], p["k0"], p["lk"], True, 128 ** -0.5,
                              2.0 ** -8 if dtype == BF16 else F)
        check((out, got[0], got[1][:2300], got[2][:2300]), val, tol)
        assert not got[1][2300:].any() and not got[2][2300:].any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("lq,lk", [([9, 5], [4, 2]), ([200, 140], [150, 30])])
@pytest.mark.parametrize("broken", [math.nan, math.inf])
def test_rows_that_see_no_key_hold_anything(dtype, lq, lk, broken):
    """causal, more queries than keys: the first queries of a sequence see nothing.  Their output and their gradient are zero and nothing
    of them enters another gradient, whatever stands in their queries and in the gradient of their output"""
    for heads in ((4, 4), (6, 2)):
        p = problem(dtype, *heads, 64, lq, lk)
        want = run(p)
        q, dout = p["q"].clone(), p["dout"].clone()
        blind = torch.zeros(q.shape[0], dtype=torch.bool, device="cuda")
        for a, n, m in zip(p["q0"], lq, lk):
            blind[a:a + n - m] = True
        q[blind], dout[blind] = broken, broken
        got = run({**p, "q": q, "dout": dout})
        assert (got[0][blind] == 0).all() and (got[1][blind] == 0).all()
        for g, w in zip(got, want):
            assert torch.equal(g, w)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("size", [1e3, 3e5, 2e7, 3e9, 1e13, 1e25])
@pytest.mark.parametrize("heads,dh,lq,lk", [
    ((4, 4), 64, [3, 9, 1], None), ((4, 2), 64, [300, 130], None), ((4, 2), 128, [300, 130], None), ((8, 2), 64, [1, 2], [3000, 1700]),
    ((2, 2), 64, [40, 30], [500, 300]), ((4, 4), 128, [3, 9, 1], None), ((2, 2), 128, [40, 30], [500, 300])])
def test_scores_of_any_size(dtype, size, heads, dh, lq, lk):
    """scores far from zero and far apart (products of powers of two: exact): each row's weight lies on its largest visible key, or in
    halves on two that are equal.  O and dV are those of one or two terms; dS is p (dP - delta), the difference of two sums of dh terms"""
    H, Hkv = heads
    p = problem(dtype, H, Hkv, dh, lq, lk, seed=8)
    g = torch.Generator().manual_seed(9)
    q, k = torch.zeros(p["q"].shape), torch.zeros(p["k"].shape)
    unit = 2.0 ** math.floor(math.log2(size) / 2)
    for sign in (1.0, -1.0):
        q[..., 5] = unit
        # heights 1 .. 1.75 in steps of 1/8 (bf16 holds them): 32 keys in a row meet each height several times
        height = torch.randint(0, 7, k.shape[:2], generator=g)
        k[..., 5] = sign * unit * (1 + height / 8.0)
        pp = {**p, "q": q.to(dtype).cuda(), "k": k.to(dtype).cuda()}
        got = [t.double().cpu() for t in run(pp, scale=1.0)]
        u = 2.0 ** -8 if dtype == BF16 else F
        V, dO, K = p["v"].double().cpu(), p["dout"].double().cpu(), k.double()
        val, eV = [torch.zeros_like(x) for x in got], torch.zeros_like(V)
        for a, n, b, m in zip(p["q0"], p["lq"], p["k0"], p["lk"]):
            seen = torch.arange(m)[None, :] <= torch.arange(n)[:, None] + (m - n)
            for h in range(H):
                at, rows, kh = slice(b, b + m), slice(a, a + n), h // (H // Hkv)
                P = torch.softmax((K[at, kh, 5] * unit).expand(n, m).masked_fill(~seen, -math.inf), 1)
                val[0][rows, h] = P @ V[at, kh]
                dP = dO[rows, h] @ V[at, kh].T
                dS = P * (dP - (dP * P).sum(1, keepdim=True))
                val[1][rows, h] = dS @ K[at, kh]
                val[2][at, kh] += dS.T @ q[rows, h].double()
                val[3][at, kh] += P.T @ dO[rows, h]
                eV[at, kh] += P.sum(0)[:, None]               # rows that lie on the key
        # p: the scores are exact; a row's sum has up to m equal terms, (m + 16) F, and p is rounded to u as an operand.  Below 2^10 a score
        # of log2 e times that size is itself rounded, by 2^-15, up to four times (m, its share in the sums of two waves, the log-sum-exp)
        rel = (max(p["lk"]) + 16) * F + u + (2.0 ** -13 if size < 1e4 else 0.0)
        D = 2 * (dO.abs().amax(2).max() * V.abs().sum(2).max())                    # at least |dP| + |delta|
        count = (H // Hkv) * max(p["lq"]) + 16
        tol = [rel * V.abs().max(), (rel + u + 4 * (dh + 16) * F) * D * 2 * unit, (rel + u + (4 * (dh + 16) + count) * F) * D * unit * eV,
               (rel + count * F) * dO.abs().max() * eV]
        for x, w, t, name in zip(got, val, tol, ("O", "dQ", "dK", "dV")):
            assert ((x - w).abs() <= u * w.abs() + t + 1e-30).all(), (name, size, sign)


# ---- nothing beyond the tensors ------------------------------------------------------------------------
GUARD = 1 << 14


class Guarded:
    """buffers of exactly the size that a C entry is told, between two zones that have to stay as they are"""

    def __init__(self):
        self.all = []

    def __call__(self, shape, dtype, fill=None):
        n = math.prod(shape) * torch.empty(0, dtype=dtype).element_size()
        buf = torch.full((n + 2 * GUARD,), 0x5A, dtype=torch.uint8, device="cuda")
        self.all.append(buf)
        view = buf[GUARD:GUARD + n].view(dtype).view(shape)
        if fill is not None:
            view.copy_(fill)
        return view

    def intact(self):
        return all((b[:GUARD] == 0x5A).all() and (b[-GUARD:] == 0x5A).all() for b in self.all)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("Tq,Tk,S,heads,dh,chunked,split", [
    (20, 20, 2, (4, 4), 64, False, False), (3, 6000, 3, (8, 2), 64, True, False), (5, 5000, 2, (4, 4), 128, True, False),
    (1500, 300, 1, (8, 1), 64, False, True), (1600, 900, 1, (12, 2), 128, False, True), (700, 900, 70, (6, 2), 24, False, False)])
def test_no_starts_make_a_kernel_leave_its_tensors(dtype, Tq, Tk, S, heads, dh, chunked, split):
    """starts and lengths of any content, through the C entries: outputs, statistics and workspaces lie between zones that stay as
    they were.  Scores of any size, with one and two planes of lse"""
    from efficientvlm_amd import _lib
    lib = _lib.load()
    H, Hkv = heads
    g = torch.Generator().manual_seed(Tq + S)
    even = lambda T: [T * i // S for i in range(S + 1)]
    wild = lambda n, T: torch.where(torch.rand(n, generator=g) < 0.3, torch.randint(-2 ** 31, 2 ** 31 - 1, (n,), generator=g),
                                    torch.randint(-9, T + 9, (n,), generator=g)).tolist()
    cases = [(even(Tq), even(Tk), None, 1.0), (even(Tq), even(Tk), wild(S, Tk), 1e6), (even(Tq), even(Tk), None, 1e12),
             ([2 ** 31 - 1, -2 ** 31] * S, [5, -7] * S, None, 1.0), ([0] + [Tq] * S, [Tk] * S + [0], None, 1.0)]
    cases += [(wild(S + 1, Tq), wild(S + 1, Tk), wild(S, Tk) if i % 2 else None, 1.0) for i in range(6)]
    for i, (cu_q, cu_k, k_lens, size) in enumerate(cases):
        print(f"case {i}", flush=True)
        i32 = lambda x: None if x is None else torch.tensor(x[:S + 1], dtype=torch.int32, device="cuda")
        cu_q, cu_k, k_lens = i32(cu_q), i32(cu_k), i32(k_lens)
        new = Guarded()
        planes = 1 + i % 2
        r = lambda *s: torch.randn(*s, generator=g) * size
        q, k, v, dout = (new(s, dtype, r(*s)) for s in ((Tq, H, dh), (Tk, Hkv, dh), (Tk, Hkv, dh), (Tq, H, dh)))
        out, lo, dq = (new((Tq, H, dh), dtype) for _ in range(3))
        dk, dv = (new((Tk, Hkv, dh), dtype) for _ in range(2))
        lse, delta = new((planes, H, Tq), F32), new((H, Tq), F32)
        a = _lib.PackedAttnArgs(dtype=_lib.BF16 if dtype == BF16 else _lib.F32, Tq=Tq, Tk=Tk, S=S, H=H, Hkv=Hkv, dh=dh, causal=i % 3 != 2,
                                scale=dh ** -0.5, lse_planes=planes, Q=q.data_ptr(), K=k.data_ptr(), V=v.data_ptr(),
                                q_tok=H * dh, q_head=dh, k_tok=Hkv * dh, k_head=dh, v_tok=Hkv * dh, v_head=dh, cu_q=cu_q.data_ptr(),
                                cu_k=cu_k.data_ptr(), k_lens=None if k_lens is None else k_lens.data_ptr(), O=out.data_ptr(),
                                O_lo=lo.data_ptr(), lse=lse.data_ptr(), dO=dout.data_ptr(), dQ=dq.data_ptr(), dK=dk.data_ptr(),
                                dV=dv.data_ptr(), do_tok=H * dh, do_head=dh, dq_tok=H * dh, dq_head=dh, dk_tok=Hkv * dh, dk_head=dh,
                                dv_tok=Hkv * dh, dv_head=dh, delta=delta.data_ptr())
        for backward, entry in ((0, lib.evlm_packed_attention_fwd), (1, lib.evlm_packed_attention_bwd)):
            n = lib.evlm_packed_attention_workspace(ctypes.byref(a), backward)
            assert (n > 0) == (split if backward else chunked)
            a.workspace = new((n,), F32).data_ptr() if n else None
            assert entry(ctypes.byref(a), torch.cuda.current_stream().cuda_stream) == 0
        torch.cuda.synchronize()
        assert new.intact(), i
        if i == 0:
            at = lambda c: c[:-1].tolist()
            n = lambda c: (c[1:] - c[:-1]).tolist()
            val, tol = definition(q, k, v, dout, at(cu_q), n(cu_q), at(cu_k), n(cu_k), True, dh ** -0.5, 2.0 ** -8 if dtype == BF16 else F)
            check((out, dq, dk, dv), val, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("heads,dh,lq,lk", [
    ((4, 4), 64, [3, 9, 30], None), ((4, 2), 64, [300, 130], None), ((4, 2), 128, [300, 130], None), ((8, 2), 64, [1, 2], [3000, 1700]),
    ((2, 2), 64, [40, 30], [500, 300]), ((6, 2), 128, [40, 30], [500, 300]), ((8, 1), 64, [1500], [300])])
def test_rows_of_small_and_large_scores_side_by_side(dtype, causal, heads, dh, lq, lk):
    """every row has a size of its own, 2^-6 .. 2^60 (scores exact, as above), so that waves hold rows near and far from zero"""
    H, Hkv = heads
    p = problem(dtype, H, Hkv, dh, lq, lk, seed=12)
    g = torch.Generator().manual_seed(13)
    q, k = torch.zeros(p["q"].shape), torch.zeros(p["k"].shape)
    q[..., 5] = 2.0 ** torch.tensor([-6, 0, 4, 9, 11, 20, 60])[torch.randint(0, 7, q.shape[:2], generator=g)]
    q[..., 5] *= torch.where(torch.rand(q.shape[:2], generator=g) < 0.5, 1.0, -1.0)
    k[..., 5] = 1 + torch.randint(0, 7, k.shape[:2], generator=g) / 8.0
    got = [t.double().cpu() for t in run({**p, "q": q.to(dtype).cuda(), "k": k.to(dtype).cuda()}, causal=causal, scale=1.0)]
    u = 2.0 ** -8 if dtype == BF16 else F
    Q, K, V, dO = q.double(), k.double(), p["v"].double().cpu(), p["dout"].double().cpu()
    val, tol = [torch.zeros_like(x) for x in got], [torch.zeros_like(x) for x in got]
    # p: sums of up to m terms, (m + 16) F; below 2^10 a score times log2 e is rounded by up to 2^-15, four times; rounded to u as an operand
    rel = (max(p["lk"]) + 16) * F + u + 2.0 ** -13
    D = 2 * (dO.abs().amax(2).max() * V.abs().sum(2).max())                        # at least |dP| + |delta|
    count = (H // Hkv) * max(p["lq"]) + 16
    err = (rel + u + (4 * (dh + 16) + count) * F) * D
    for a, n, b, m in zip(p["q0"], p["lq"], p["k0"], p["lk"]):
        seen = torch.ones(n, m, dtype=torch.bool)
        if causal:
            seen = torch.arange(m)[None, :] <= torch.arange(n)[:, None] + (m - n)
        for h in range(H):
            at, rows, kh = slice(b, b + m), slice(a, a + n), h // (H // Hkv)
            P = torch.softmax((Q[rows, h, 5][:, None] * K[at, kh, 5]).masked_fill(~seen, -math.inf), 1).nan_to_num(0.0)
            dP = dO[rows, h] @ V[at, kh].T
            dS = P * (dP - (dP * P).sum(1, keepdim=True))
            val[0][rows, h], val[1][rows, h] = P @ V[at, kh], dS @ K[at, kh]
            val[2][at, kh] += dS.T @ Q[rows, h]
            val[3][at, kh] += P.T @ dO[rows, h]
            tol[0][rows, h], tol[1][rows, h] = rel * V.abs().max(), err * 2
            tol[2][at, kh] += err * (P.T @ Q[rows, h].abs())
            tol[3][at, kh] += (rel + count * F) * (P.T @ dO[rows, h].abs())
    for x, w, t, name in zip(got, val, tol, ("O", "dQ", "dK", "dV")):
        assert ((x - w).abs() <= u * w.abs() + t + 1e-30).all(), name
