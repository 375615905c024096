"""The serving operators on the GPU against plain 64-bit implementations: kv_append (paged cache
with the position rotation), attention_varlen (packed prompts, grouped heads, causal) and
attention_paged (one token per sequence), alone and as a prompt followed by single tokens.

Tolerances, per element, from the operators' arithmetic.  u = eps / 2 of the storage type.
- A rotated element is two f32 products and a sum rounded once: u |y| + 2^-22 (|x c| + |x' s|),
  and half the smallest f16 subnormal, 2^-25.
- An attention output is sum w_j v_j / sum w_j with weights rounded to the storage type in the
  first sum, or in both (relative u each), exponentials good to 1e-4 (cubic of the FMA pipe: 8.3e-5) and
  exponents s c wrong by at most |s c| 2^-22 + D 2^-23 sum_e |q_e k_e| c, which max |s| <= 64 keeps
  below 2^-9 for the inputs here (|q.k| scale <= 16 with unit normals).  A weight's relative
  error e moves the output by at most e sum w_j |v_j - o| / sum w_j <= 2 e A with A = sum w_j |v_j|
  / sum w_j; f16 weights below 2^-14 are subnormal, wrong by 2^-25 each.  The result is rounded once."""
from __future__ import annotations

import math

import pytest
import torch

from headshot_b200._lib import HS_ERR_INVALID, HS_ERR_TIMEOUT, HsError
from headshot_b200.engine import GpuContext, PagedKv, Rope

pytestmark = pytest.mark.gpu
TORCH = {"bf16": torch.bfloat16, "f16": torch.float16}
SHAPES = [(4, 4, 64), (8, 2, 64), (3, 1, 64), (10, 2, 64), (4, 4, 128), (8, 2, 128), (7, 1, 128), (32, 1, 128)]


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def normal(g, *shape, dtype="bf16"):
    return torch.randn(shape, generator=g, device="cuda").to(TORCH[dtype])


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def offsets(lens):
    at = [0]
    for n in lens:
        at.append(at[-1] + n)
    return ints(at)


def attend64(q, k, v, first_limit, causal, scale=None):
    """q (m, hq, d), k, v (n, hkv, d) -> (out, A) in 64 bits; query i sees keys j <= first_limit + i."""
    m, hq, d = q.shape
    n, hkv = k.shape[:2]
    qd = q.double().reshape(m, hkv, hq // hkv, d).permute(1, 2, 0, 3)
    kd, vd = k.double().permute(1, 0, 2)[:, None], v.double().permute(1, 0, 2)[:, None]
    s = qd @ kd.transpose(-1, -2) * (scale or d ** -0.5)
    if causal:
        i = torch.arange(m, device=q.device)[:, None] + first_limit
        s = s.masked_fill(torch.arange(n, device=q.device) > i, -math.inf)
    w = torch.exp(s - s.amax(-1, keepdim=True).clamp_min(-1e30)) if n else s
    tot = w.sum(-1, keepdim=True)
    w = torch.where(tot > 0, w / tot.clamp_min(1e-300), torch.zeros_like(w))
    back = lambda x: x.permute(2, 0, 1, 3).reshape(m, hq, d)  # noqa: E731
    return back(w @ vd), back(w @ vd.abs())


def check_attention(got, ref, a, keys, dtype, vmax):
    u = torch.finfo(TORCH[dtype]).eps / 2
    tol = u * ref.abs() + 2 * (u + 1e-4 + 2.0 ** -9 * 0.1) * a + 1e-30
    if dtype == "f16":
        tol = tol + 2.0 ** -25 * (1 + keys * vmax)
    assert torch.isfinite(got).all()
    over = ((got.double() - ref).abs() - tol).max().item()
    assert over <= 0, f"past the tolerance by {over}"


def packed_check(out, q, k, v, qlens, klens, causal, dtype, scale=None):
    q0 = k0 = 0
    for a, b in zip(qlens, klens):
        if a:
            for i0 in range(0, a, 512):  # bounds the 64-bit scores
                i1 = min(a, i0 + 512)
                ref, mass = attend64(q[q0 + i0:q0 + i1], k[k0:k0 + b], v[k0:k0 + b], b - a + i0, causal, scale)
                vmax = v[k0:k0 + b].abs().max().item() if b else 0.0
                check_attention(out[q0 + i0:q0 + i1], ref, mass, b, dtype, vmax)
        q0, k0 = q0 + a, k0 + b


# ---------------------------------------------------------------- kv_append --


def tables(rows, d, seed):
    g = gen(seed)
    a = torch.rand(rows, d, generator=g, device="cuda", dtype=torch.float64) * 6.3  # halves differ on purpose
    return a.sin().float(), a.cos().float()


def table_for(lens, page, g, spare=3):
    need = [max(0, -(-n // page)) for n in lens]
    pool = sum(need) + spare
    order = torch.randperm(pool, generator=g, device="cuda").to(torch.int32)
    t = torch.full((len(lens), max(1, max(need))), -1, dtype=torch.int32, device="cuda")
    at = 0
    for s, n in enumerate(need):
        t[s, :n] = order[at:at + n]
        at += n
    return t, pool


def append_reference(x, pos, rope, u):
    """Rotated rows in 64 bits and the tolerance of each element."""
    y, tol = x.double(), torch.zeros_like(x, dtype=torch.float64)
    if rope is not None:
        d = x.shape[-1]
        f = pos if rope.tokens_per_frame is None else pos % rope.tokens_per_frame
        r = f - rope.prefix
        on = (r >= 0)[:, None, None]
        c, s = rope.cos.double()[r.clamp_min(0)][:, None], rope.sin.double()[r.clamp_min(0)][:, None]
        other = torch.cat([-y[..., d // 2:], y[..., :d // 2]], -1)
        z = y * c + other * s
        tol = torch.where(on, u * z.abs() + 2.0 ** -22 * ((y * c).abs() + (other * s).abs()) + 2.0 ** -25, tol)
        y = torch.where(on, z, y)
    return y, tol


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("hq,hkv,d", SHAPES)
@pytest.mark.parametrize("page,new,old,rope", [
    (16, [1, 1, 1], [0, 15, 16], "text"),
    (1, [3, 1, 5], [0, 2, 7], "none"),
    (5, [7, 0, 33, 1], [4, 9, 0, 0], "frames"),
    (100, [250, 1, 99], [0, 99, 1], "text"),
    (64, [1], [500], "frames"),
])
def test_kv_append(gpu_ctx, dtype, hq, hkv, d, page, new, old, rope):
    g = gen(hash((hq, hkv, d, page)) % 1000)
    n, pad = sum(new), 3
    lens = [a + b for a, b in zip(new, old)]
    table, pool = table_for(lens, page, g)
    kc, vc = (normal(g, pool, hkv, page, d, dtype=dtype) for _ in range(2))
    rp = None
    if rope != "none":
        rows = max(lens) if rope == "text" else 20
        sin, cos = tables(rows, d, 7)
        rp = Rope(sin, cos, 0) if rope == "text" else Rope(sin, cos, 4, 24)
    single = all(a == 1 for a in new)
    proj = normal(g, n if single else n + pad, hq + 2 * hkv, d, dtype=dtype)  # padding rows behind the last sequence
    q, k, v = proj[:, :hq], proj[:, hq:hq + hkv], proj[:, hq + hkv:]
    q_out, k_out = torch.full_like(q, 9).contiguous(), torch.full_like(k, 9).contiguous()
    k0, v0 = kc.clone(), vc.clone()
    got = gpu_ctx.kv_append(PagedKv(kc, vc, table), k, v, ints(lens), cu_new=None if single else offsets(new), rope=rp,
                            q=q, q_out=q_out, k_out=k_out)
    gpu_ctx.sync()
    assert got is q_out
    seq = torch.repeat_interleave(torch.arange(len(new), device="cuda"), torch.tensor(new, device="cuda"))
    pos = torch.cat([torch.arange(b, b + a, device="cuda") for a, b in zip(new, old)])
    u = torch.finfo(TORCH[dtype]).eps / 2
    for x, y in ((q, q_out), (k, k_out)):
        ref, tol = append_reference(x[:n], pos, rp, u)
        assert ((y[:n].double() - ref).abs() <= tol).all()
        assert (y[n:] == 9).all()
    at, off = table[seq, pos // page].long(), pos % page
    k0[at, :, off], v0[at, :, off] = k_out[:n], v[:n]
    assert torch.equal(kc, k0) and torch.equal(vc, v0)  # every other row as it was


def test_kv_append_in_place_and_without_queries(gpu_ctx):
    g = gen(3)
    table, pool = table_for([40, 9], 16, g)
    sin, cos = tables(40, 64, 1)
    rope = Rope(sin, cos, 0)
    k, v, q = normal(g, 49, 2, 64), normal(g, 49, 2, 64), normal(g, 49, 6, 64)
    cu, lens = offsets([40, 9]), ints([40, 9])
    caches = [PagedKv(torch.zeros(pool, 2, 16, 64, dtype=torch.bfloat16, device="cuda"),
                      torch.zeros(pool, 2, 16, 64, dtype=torch.bfloat16, device="cuda"), table) for _ in range(2)]
    k_rot = torch.empty_like(k)
    q_rot = gpu_ctx.kv_append(caches[0], k, v, lens, cu, rope, q=q, k_out=k_rot)
    assert gpu_ctx.kv_append(caches[1], k, v, lens, cu, rope) is None
    assert torch.equal(caches[0].k, caches[1].k) and torch.equal(caches[0].v, caches[1].v)
    q2, k2 = q.clone(), k.clone()
    assert gpu_ctx.kv_append(caches[1], k2, v, lens, cu, rope, q=q2, q_out=q2, k_out=k2) is q2
    gpu_ctx.sync()
    assert torch.equal(q2, q_rot) and torch.equal(k2, k_rot) and torch.equal(caches[0].k, caches[1].k)


def test_kv_append_many_sequences_find_their_tokens(gpu_ctx):
    """Offsets past one and two 32-way search steps, empty sequences among them."""
    for n_seqs in (1, 31, 33, 1000, 1100):
        g = gen(n_seqs)
        new = torch.randint(0, 4, (n_seqs,), generator=g, device="cuda").tolist()
        new[-1] = 2
        n = sum(new)
        table = torch.arange(n_seqs, device="cuda", dtype=torch.int32)[:, None].contiguous()
        kc, vc = (torch.zeros(n_seqs, 1, 4, 64, dtype=torch.float16, device="cuda") for _ in range(2))
        k, v = normal(g, n, 1, 64, dtype="f16"), normal(g, n, 1, 64, dtype="f16")
        gpu_ctx.kv_append(PagedKv(kc, vc, table), k, v, ints(new), cu_new=offsets(new))
        gpu_ctx.sync()
        want = torch.zeros_like(kc)
        seq = torch.repeat_interleave(torch.arange(n_seqs, device="cuda"), torch.tensor(new, device="cuda"))
        i = torch.cat([torch.arange(a, device="cuda") for a in new])
        want[seq, :, i] = k
        assert torch.equal(kc, want)


def test_kv_append_padding_sequences(gpu_ctx):
    """kv_lens of 0 (an idle slot of a batch) leaves the token alone."""
    g = gen(4)
    kc, vc = normal(g, 4, 2, 16, 64), normal(g, 4, 2, 16, 64)
    k0, v0 = kc.clone(), vc.clone()
    table = ints([[0], [-1], [2]])
    k, v, q = normal(g, 3, 2, 64), normal(g, 3, 2, 64), normal(g, 3, 4, 64)
    q_out = torch.full_like(q, 5)
    gpu_ctx.kv_append(PagedKv(kc, vc, table), k, v, ints([1, 0, 7]), q=q, q_out=q_out)
    gpu_ctx.sync()
    k0[0, :, 0], v0[0, :, 0], k0[2, :, 6], v0[2, :, 6] = k[0], v[0], k[2], v[2]
    assert torch.equal(kc, k0) and torch.equal(vc, v0)
    assert torch.equal(q_out[0], q[0]) and (q_out[1] == 5).all() and torch.equal(q_out[2], q[2])


# --------------------------------------------------------- attention_varlen --

LENGTHS = [
    ([1], None),
    ([17], None),
    ([128, 129], None),
    ([64, 1, 300, 7, 0, 191, 257], None),
    ([1000, 3], None),
    ([5, 40, 130], [300, 40, 131]),     # behind keys that are there already
    ([40, 3, 200], [8, 0, 190]),        # queries that see nothing, a sequence without keys
]


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("hq,hkv,d", SHAPES)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("qlens,klens", LENGTHS)
def test_varlen(gpu_ctx, dtype, hq, hkv, d, causal, qlens, klens):
    g = gen(len(qlens) * 100 + hq + d)
    nq, nk = sum(qlens), sum(klens or qlens)
    pad = 0 if klens is None else 5
    q = normal(g, nq + pad, hq, d, dtype=dtype)
    k, v = normal(g, nk + pad, hkv, d, dtype=dtype), normal(g, nk + pad, hkv, d, dtype=dtype)
    k[nk:], v[nk:] = math.nan, math.inf  # behind the last sequence
    out = torch.full_like(q, 3)
    gpu_ctx.attention_varlen(q, k, v, offsets(qlens), cu_k=None if klens is None else offsets(klens), causal=causal,
                             out=out)
    gpu_ctx.sync()
    packed_check(out, q, k, v, qlens, klens or qlens, causal, dtype)
    assert (out[nq:] == 3).all()


@pytest.mark.parametrize("hq,hkv,d", [(4, 2, 64), (4, 2, 128)])
def test_varlen_reads_a_fused_projection_in_place(gpu_ctx, hq, hkv, d):
    g = gen(8)
    lens = [70, 200, 31]
    rows = normal(g, sum(lens), hq + 2 * hkv + 1, d)
    q, k, v = rows[:, :hq], rows[:, hq:hq + hkv], rows[:, hq + hkv:hq + 2 * hkv]
    out = gpu_ctx.attention_varlen(q, k, v, offsets(lens), scale=0.3)
    gpu_ctx.sync()
    packed_check(out, q, k, v, lens, lens, True, "bf16", 0.3)


@pytest.mark.parametrize("d", [64, 128])
def test_varlen_neighbours_do_not_leak(gpu_ctx, d):
    """Infinities and NaN in the next sequence, inside the same key tile."""
    g = gen(9)
    lens = [50, 45, 100, 13]
    q, k, v = normal(g, 208, 4, d), normal(g, 208, 4, d), normal(g, 208, 4, d)
    k[50:95], v[50:95] = math.nan, math.nan
    k[195:], v[195:] = math.inf, -math.inf
    for causal in (True, False):
        out = gpu_ctx.attention_varlen(q, k, v, offsets(lens), causal=causal)
        gpu_ctx.sync()
        packed_check(out[:50], q[:50], k[:50], v[:50], [50], [50], causal, "bf16")
        packed_check(out[95:195], q[95:195], k[95:195], v[95:195], [100], [100], causal, "bf16")
        assert out[50:95].isnan().all()


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("d", [64, 128])
def test_varlen_rising_and_extreme_scores(gpu_ctx, dtype, d):
    """A maximum that moves with every key tile, and scores far below zero."""
    g = gen(10)
    n = 700
    q = torch.ones(n, 2, d, device="cuda") * 0.5
    k = torch.linspace(-8, 8, n, device="cuda")[:, None, None].expand(n, 2, d) * torch.tensor([1.0, -1.0], device="cuda")[:, None]
    q, k = q.to(TORCH[dtype]), k.contiguous().to(TORCH[dtype])
    v = normal(g, n, 2, d, dtype=dtype)
    out = gpu_ctx.attention_varlen(q, k, v, offsets([n]))
    gpu_ctx.sync()
    packed_check(out, q, k, v, [n], [n], True, dtype)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("d", [64, 128])
def test_largest_values_in_masked_places(gpu_ctx, dtype, d):
    """The type's largest values behind a causal mask, and on keys whose score lies 200 binades down,
    add nothing: their weights are zero, not tiny (2^-125 of bf16's largest value would be 8)."""
    g = gen(17)
    n, big = 200, torch.finfo(TORCH[dtype]).max
    q, k, v = normal(g, n, 2, d, dtype=dtype), normal(g, n, 2, d, dtype=dtype), normal(g, n, 2, d, dtype=dtype)
    v[120:] = big
    k[120:] = -big / 1e30 if dtype == "bf16" else -big
    out = gpu_ctx.attention_varlen(q, k, v, offsets([n]))
    gpu_ctx.sync()
    packed_check(out[:120], q[:120], k[:120], v[:120], [120], [120], True, dtype)

    # Far below the maximum: queries of ones, keys of +-c with |q.k| scale log2 e = 100 each way.
    one = torch.ones(n, 2, d, device="cuda").to(TORCH[dtype])
    c = 100.0 / (d ** 0.5 * 1.4426950408889634)
    low = torch.full_like(one, c)
    low[1::3] = -c  # 200 binades below the others
    w = normal(g, n, 2, d, dtype=dtype)
    w[1::3] = big
    for causal in (True, False):
        out = gpu_ctx.attention_varlen(one, low, w, offsets([n]), causal=causal)
        keep = [i for i in range(n) if i % 3 != 1]
        gpu_ctx.sync()
        for i in (0, 1, 5, 63, 64, 150, 199):
            seen = [j for j in keep if not causal or j <= i]
            want = w[seen].double().mean(0)
            mass = w[seen].double().abs().mean(0)
            check_attention(out[i], want, mass, n, dtype, w[seen].abs().max().item())


@pytest.mark.parametrize("dtype,size", [("bf16", 300.0), ("bf16", 2e3), ("bf16", 1e9), ("f16", 2e3), ("f16", 6e4)])
@pytest.mark.parametrize("d", [64, 128])
def test_huge_scores(gpu_ctx, dtype, size, d):
    """Scores whose product with the scale rounds away whole binades: each row still belongs to its
    largest score, which the inputs set apart from the others by far.  (Packed prompts: to 2^26.)"""
    g = gen(18)
    n = 130
    sign = torch.where(torch.rand(n, 1, d, generator=g, device="cuda") < 0.5, -1.0, 1.0)
    k = (sign * size).to(TORCH[dtype])
    q = (sign.flip(0) * size).to(TORCH[dtype])
    v = normal(g, n, 1, d, dtype=dtype)
    if size * size * d ** 0.5 <= 2.0 ** 26:
        out = gpu_ctx.attention_varlen(q, k, v, offsets([n]), causal=False)
    else:
        out = v.flip(0)
    table = torch.arange(9, dtype=torch.int32, device="cuda")[None]
    kc, vc = (torch.zeros(9, 1, 16, d, dtype=TORCH[dtype], device="cuda") for _ in range(2))
    cache = PagedKv(kc, vc, table)
    gpu_ctx.kv_append(cache, k, v, ints([n]), cu_new=offsets([n]))
    rows = [gpu_ctx.attention_paged(q[i:i + 1], cache, ints([n])) for i in (0, 40, 129)]
    gpu_ctx.sync()
    # Row i's own sign pattern is key n - 1 - i: score d size^2, the next one at least 2 size^2 less.
    # Its weight is 2^r with r the rounding of the maximum times the scale, |r| <= 2 here, so not
    # 1: it is rounded (u) where it multiplies the value and not in the sum, hence no equality.
    check_attention(out, v.flip(0).double(), v.flip(0).double().abs(), n, dtype, v.abs().max().item())
    for i, got in zip((0, 40, 129), rows):
        assert torch.equal(got[0], v[n - 1 - i])


def test_varlen_long(gpu_ctx):
    """Many key tiles and items per processor, ragged, against 64 bits on sampled rows."""
    g = gen(11)
    lens = [9001, 4, 2600]
    q, k, v = normal(g, sum(lens), 8, 128), normal(g, sum(lens), 2, 128), normal(g, sum(lens), 2, 128)
    out = gpu_ctx.attention_varlen(q, k, v, offsets(lens))
    again = gpu_ctx.attention_varlen(q, k, v, offsets(lens))
    gpu_ctx.sync()
    assert torch.equal(out, again)
    for i in (0, 1, 127, 128, 5000, 9000):
        ref, a = attend64(q[i:i + 1], k[:i + 1], v[:i + 1], i, True)
        check_attention(out[i:i + 1], ref, a, i + 1, "bf16", 6.0)
    packed_check(out[9001:], q[9001:], k[9001:], v[9001:], lens[1:], lens[1:], True, "bf16")


@pytest.mark.parametrize("d", [64, 128])
def test_varlen_output_aligned_to_16_bytes_only(gpu_ctx, d):
    g = gen(16)
    lens = [130, 7]
    q, k, v = normal(g, 137, 6, d), normal(g, 137, 2, d), normal(g, 137, 2, d)
    buf = torch.full((137 * 6 * d + 16,), 2.0, dtype=torch.bfloat16, device="cuda")
    out = buf[8:8 + 137 * 6 * d].view(137, 6, d)
    assert out.data_ptr() % 32 == 16
    gpu_ctx.attention_varlen(q, k, v, offsets(lens), out=out)
    want = gpu_ctx.attention_varlen(q, k, v, offsets(lens))
    gpu_ctx.sync()
    assert torch.equal(out, want) and (buf[:8] == 2).all() and (buf[-8:] == 2).all()


def test_varlen_many_sequences(gpu_ctx):
    """More sequences than the scheduler scans at once, empty ones and every length class among them."""
    for n_seqs, longest, causal in ((33, 700, True), (1500, 5, True), (200, 300, False)):
        g = gen(n_seqs)
        qlens = torch.randint(0, longest + 1, (n_seqs,), generator=g, device="cuda").tolist()
        extra = torch.randint(0, 60, (n_seqs,), generator=g, device="cuda").tolist()
        klens = [max(0, a + b - 20) for a, b in zip(qlens, extra)]
        q = normal(g, sum(qlens), 4, 64)
        k, v = normal(g, sum(klens), 2, 64), normal(g, sum(klens), 2, 64)
        out = gpu_ctx.attention_varlen(q, k, v, offsets(qlens), cu_k=offsets(klens), causal=causal)
        gpu_ctx.sync()
        packed_check(out, q, k, v, qlens, klens, causal, "bf16")


@pytest.mark.parametrize("hq,hkv", [(128, 1), (100, 1), (96, 2), (1, 1)])
@pytest.mark.parametrize("d", [64, 128])
def test_varlen_group_extremes(gpu_ctx, hq, hkv, d):
    g = gen(hq)
    lens = [3, 77, 200]
    q, k, v = normal(g, 280, hq, d), normal(g, 280, hkv, d), normal(g, 280, hkv, d)
    out = gpu_ctx.attention_varlen(q, k, v, offsets(lens))
    gpu_ctx.sync()
    packed_check(out, q, k, v, lens, lens, True, "bf16")


def test_varlen_no_keys_at_all(gpu_ctx):
    q = normal(gen(14), 70, 4, 128)
    none = q[:0, :2]
    for causal in (True, False):
        out = gpu_ctx.attention_varlen(q, none, none, offsets([30, 40]), cu_k=offsets([0, 0]), causal=causal)
        gpu_ctx.sync()
        assert (out == 0).all()


def test_nan_query_stays_in_its_row(gpu_ctx):
    g = gen(15)
    q, k, v = normal(g, 300, 4, 64), normal(g, 300, 2, 64), normal(g, 300, 2, 64)
    clean = gpu_ctx.attention_varlen(q, k, v, offsets([300]))
    q[123, 2] = math.nan
    out = gpu_ctx.attention_varlen(q, k, v, offsets([300]))
    lens = [900, 40]
    p, cache = paged_case(g, 8, 2, 128, 16, lens, "f16")
    p_clean = gpu_ctx.attention_paged(p, cache, ints(lens))
    p[0, 5] = math.nan
    p_out = gpu_ctx.attention_paged(p, cache, ints(lens))
    gpu_ctx.sync()
    assert out[123, 2].isnan().all() and p_out[0, 5].isnan().all()
    out[123, 2], p_out[0, 5] = clean[123, 2], p_clean[0, 5]
    assert torch.equal(out, clean) and torch.equal(p_out, p_clean)


def test_varlen_bad_offsets_are_reported(gpu_ctx):
    g = gen(12)
    q, k, v = normal(g, 40, 4, 64), normal(g, 40, 4, 64), normal(g, 40, 4, 64)
    good = gpu_ctx.attention_varlen(q, k, v, offsets([20, 20]))
    for cu in ([0, 20, 60], [0, 30, 20], [0, -5, 40]):
        gpu_ctx.attention_varlen(q, k, v, ints(cu))
        with pytest.raises(HsError) as e:
            gpu_ctx.sync()
        assert e.value.status == HS_ERR_INVALID and "offsets" in e.value.message
    again = gpu_ctx.attention_varlen(q, k, v, offsets([20, 20]))
    gpu_ctx.sync()
    assert torch.equal(good, again)


def test_varlen_timeout_is_reported_and_leaves_the_context_usable():
    """Wait bound 0: every in-kernel wait that has to wait gives up at once (no fault, no hang)."""
    ctx = GpuContext(0)
    g = gen(13)
    lens = [900, 300]
    for d in (64, 128):
        q, k, v = (normal(g, 1200, h, d) for h in (8, 2, 2))
        good = ctx.attention_varlen(q, k, v, offsets(lens))
        ctx.sync()
        ctx.set_wait_timeout_ms(0)
        ctx.attention_varlen(q, k, v, offsets(lens))
        with pytest.raises(HsError) as e:
            ctx.sync()
        assert e.value.status == HS_ERR_TIMEOUT
        ctx.set_wait_timeout_ms(2000)
        again = ctx.attention_varlen(q, k, v, offsets(lens))
        ctx.sync()
        assert torch.equal(good, again)
    ctx.close()


# ---------------------------------------------------------- attention_paged --


def paged_case(g, hq, hkv, d, page, lens, dtype):
    table, pool = table_for(lens, page, g)
    q = normal(g, len(lens), hq, d, dtype=dtype)
    kc, vc = (normal(g, pool, hkv, page, d, dtype=dtype) for _ in range(2))
    return q, PagedKv(kc, vc, table)


def gathered(cache, s, n):
    page = cache.k.shape[2]
    p = torch.arange(max(n, 0), device="cuda")
    at, off = cache.block_table[s][p // page].long(), p % page
    return cache.k[at, :, off], cache.v[at, :, off]


def paged_check(out, q, cache, lens, dtype, scale=None):
    for s, n in enumerate(lens):
        if n <= 0:
            assert (out[s] == 0).all()
            continue
        k, v = gathered(cache, s, n)
        ref, a = attend64(q[s:s + 1], k, v, n - 1, False, scale)
        check_attention(out[s:s + 1], ref, a, n, dtype, v.abs().max().item())


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("hq,hkv,d", SHAPES)
@pytest.mark.parametrize("page,lens", [
    (16, [1]),
    (16, [0, 1, 15, 16, 17, 500]),
    (1, [3, 70]),
    (5, [63, 64, 65, 1000, 0]),
    (24, [129, 2]),
    (100, [99, 100, 101, 777]),
    (64, [5000]),
    (256, [4099, 1, 300]),
    (8, [37, 1000]),
    (12, [11, 12, 13, 600]),
])
def test_paged(gpu_ctx, dtype, hq, hkv, d, page, lens):
    g = gen(page + hq + d)
    q, cache = paged_case(g, hq, hkv, d, page, lens, dtype)
    # what lies behind the last token of a sequence's last page must not matter
    for s, n in enumerate(lens):
        if n % page:
            at = cache.block_table[s, n // page].long()
            cache.k[at, :, n % page:], cache.v[at, :, n % page:] = math.nan, math.inf
    out = gpu_ctx.attention_paged(q, cache, ints(lens))
    again = gpu_ctx.attention_paged(q, cache, ints(lens))
    gpu_ctx.sync()
    assert torch.equal(out, again)
    paged_check(out, q, cache, lens, dtype)


def test_paged_many_sequences_one_workspace(gpu_ctx):
    """Ragged batches of several shapes through one workspace, which each call leaves ready."""
    ws = gpu_ctx.paged_workspace()
    before = ws.clone()
    for seqs, longest, hq, hkv, d in ((300, 40, 4, 2, 64), (37, 3001, 8, 8, 64), (2, 20001, 8, 1, 128), (700, 9, 2, 1, 128)):
        g = gen(seqs)
        lens = torch.randint(0, longest + 1, (seqs,), generator=g, device="cuda").tolist()
        lens[0], lens[-1] = 0, longest
        q, cache = paged_case(g, hq, hkv, d, 16, lens, "bf16")
        out = gpu_ctx.attention_paged(q, cache, ints(lens), workspace=ws)
        gpu_ctx.sync()
        paged_check(out, q, cache, lens, "bf16")
    assert before.numel() == ws.numel()


def test_paged_idle_slots_and_thousands_of_sequences(gpu_ctx):
    g = gen(25)
    lens = torch.randint(0, 30, (5000,), generator=g, device="cuda").tolist()
    q, cache = paged_case(g, 2, 1, 64, 16, lens, "bf16")
    given = [-7 if n == 0 else n for n in lens]  # any length below one is an idle slot
    out = gpu_ctx.attention_paged(q, cache, ints(given))
    gpu_ctx.sync()
    paged_check(out[:300], q[:300], cache, lens[:300], "bf16")
    paged_check(out[-100:], q[-100:], PagedKv(cache.k, cache.v, cache.block_table[-100:]), lens[-100:], "bf16")
    assert (out[[i for i, n in enumerate(lens) if n == 0]] == 0).all()


@pytest.mark.parametrize("hq,hkv", [(48, 1), (17, 1), (128, 2)])
@pytest.mark.parametrize("d", [64, 128])
def test_paged_more_heads_than_one_tile(gpu_ctx, hq, hkv, d):
    g = gen(hq + d)
    lens = [2000, 5, 64]
    q, cache = paged_case(g, hq, hkv, d, 32, lens, "bf16")
    out = gpu_ctx.attention_paged(q, cache, ints(lens))
    gpu_ctx.sync()
    paged_check(out, q, cache, lens, "bf16")


def test_paged_strided_queries_and_scale(gpu_ctx):
    g = gen(21)
    lens = [33, 900, 7]
    q, cache = paged_case(g, 6, 2, 128, 32, lens, "f16")
    wide = normal(g, 3, 9, 128, dtype="f16")
    out = torch.empty(3, 6, 128, dtype=torch.float16, device="cuda")
    assert gpu_ctx.attention_paged(wide[:, :6], cache, ints(lens), scale=0.25, out=out) is out
    gpu_ctx.sync()
    paged_check(out, wide[:, :6], cache, lens, "f16", 0.25)


@pytest.mark.parametrize("d", [64, 128])
def test_paged_rising_scores(gpu_ctx, d):
    g = gen(22)
    lens = [3000]
    q, cache = paged_case(g, 2, 1, d, 16, lens, "bf16")
    q[:, 0], q[:, 1] = 0.5, -0.5
    up = torch.linspace(-8, 8, 3000, device="cuda").to(torch.bfloat16)
    p = torch.arange(3000, device="cuda")
    cache.k[cache.block_table[0][p // 16].long(), :, p % 16] = up[:, None, None].expand(3000, 1, d)
    out = gpu_ctx.attention_paged(q, cache, ints(lens))
    gpu_ctx.sync()
    paged_check(out, q, cache, lens, "bf16")


def test_paged_offsets_past_32_bits(gpu_ctx):
    """Pages whose element offset (2^32 and more) does not fit 32 bits."""
    page, hkv, d = 256, 8, 128
    pool = (1 << 32) // (page * hkv * d) + 8
    kc, vc = (torch.empty(pool, hkv, page, d, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    g = gen(23)
    use = [pool - 1, 0, pool - 3, (1 << 31) // (page * hkv * d)]
    for p in use:
        kc[p], vc[p] = normal(g, hkv, page, d), normal(g, hkv, page, d)
    cache = PagedKv(kc, vc, ints([use]))
    lens = ints([3 * page + 40])
    k, v, q = normal(g, 1, hkv, d), normal(g, 1, hkv, d), normal(g, 1, 16, d)
    gpu_ctx.kv_append(cache, k, v, lens)
    out = gpu_ctx.attention_paged(q, cache, lens)
    gpu_ctx.sync()
    assert torch.equal(kc[use[3], :, 39], k[0]) and torch.equal(vc[use[3], :, 39], v[0])
    paged_check(out, q, cache, [3 * page + 40], "bf16")


def test_bad_pages_lengths_and_positions_are_reported(gpu_ctx):
    """An index outside its tensors is skipped and reported; the other sequences are unharmed."""
    g = gen(24)
    lens = [40, 40, 40]
    q, cache = paged_case(g, 4, 2, 64, 16, lens, "bf16")
    good = gpu_ctx.attention_paged(q, cache, ints(lens))
    gpu_ctx.sync()
    pool = cache.k.shape[0]
    for bad in (-1, pool, 2 ** 31 - 1):
        table = cache.block_table.clone()
        table[1, 1] = bad
        out = gpu_ctx.attention_paged(q, PagedKv(cache.k, cache.v, table), ints(lens))
        with pytest.raises(HsError) as e:
            gpu_ctx.sync()
        assert e.value.status == HS_ERR_INVALID and "page" in e.value.message
        assert torch.equal(out[[0, 2]], good[[0, 2]])
    out = gpu_ctx.attention_paged(q, cache, ints([40, 49, 40]))  # three pages of 16
    with pytest.raises(HsError) as e:
        gpu_ctx.sync()
    assert e.value.status == HS_ERR_INVALID and "length" in e.value.message
    assert torch.equal(out[[0, 2]], good[[0, 2]])

    k, v = normal(g, 3, 2, 64), normal(g, 3, 2, 64)
    for table_bad, kv_lens, rope, word in ((True, [40, 40, 40], None, "page"), (False, [40, 49, 40], None, "length"),
                                           (False, [30, 40, 30], Rope(*tables(30, 64, 2), 0), "rotation")):
        kc, vc = cache.k.clone(), cache.v.clone()
        table = cache.block_table.clone()
        if table_bad:
            table[1, 2] = pool
        gpu_ctx.kv_append(PagedKv(kc, vc, table), k, v, ints(kv_lens), rope=rope)
        with pytest.raises(HsError) as e:
            gpu_ctx.sync()
        assert e.value.status == HS_ERR_INVALID and word in e.value.message
        vc[cache.block_table[0, (kv_lens[0] - 1) // 16].long(), :, (kv_lens[0] - 1) % 16] -= v[0]
        changed = (vc != cache.v).any(-1).any(1).sum().item()
        assert changed <= 2  # rows of sequences 0 and 2 only
    gpu_ctx.sync()


# ------------------------------------------------------------------ refusals --


def test_refusals_of_the_library(gpu_ctx):
    g = gen(30)
    q, cache = paged_case(g, 4, 2, 64, 16, [20, 20], "bf16")
    lens = ints([20, 20])
    ws = gpu_ctx.paged_workspace()
    f32 = PagedKv(cache.k.float(), cache.v.float(), cache.block_table)
    odd = torch.zeros(2 * 4 * 64 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(2, 4, 64)  # 2-byte aligned
    k96 = torch.zeros(2, 2, 16, 96, dtype=torch.bfloat16, device="cuda")
    calls = [
        lambda: gpu_ctx.attention_paged(q.float(), f32, lens),
        lambda: gpu_ctx.attention_paged(odd, cache, lens),
        lambda: gpu_ctx.attention_paged(q, cache, lens, workspace=ws[:-16]),
        lambda: gpu_ctx.attention_paged(q[:, :, :1].expand(2, 4, 64).contiguous()[..., :0].expand(2, 4, 0), cache, lens),
        lambda: gpu_ctx.attention_paged(torch.zeros(2, 4, 96, dtype=torch.bfloat16, device="cuda"),
                                        PagedKv(k96, k96, cache.block_table), lens),
        lambda: gpu_ctx.attention_varlen(odd, odd, odd, offsets([2])),
        lambda: gpu_ctx.attention_varlen(torch.zeros(2, 129, 64, dtype=torch.bfloat16, device="cuda"),
                                         torch.zeros(2, 1, 64, dtype=torch.bfloat16, device="cuda"),
                                         torch.zeros(2, 1, 64, dtype=torch.bfloat16, device="cuda"), offsets([2])),
        lambda: gpu_ctx.kv_append(cache, odd[:, :2], odd[:, 2:], lens),
        lambda: gpu_ctx.kv_append(cache, normal(g, 2, 2, 64), normal(g, 2, 2, 64), lens,
                                  rope=Rope(*tables(10, 64, 1), 5, 24)),  # 19 rows needed
    ]
    for i, call in enumerate(calls):
        with pytest.raises((HsError, AssertionError)):
            call()
    gpu_ctx.sync()


# ------------------------------------------------------------- used together --


def test_prompt_then_tokens(gpu_ctx):
    """Prompts of three lengths enter the cache, then twenty single tokens each: every output against
    64-bit attention over everything before it, rotated in 64 bits from the stored projections."""
    hq, hkv, d, page = 8, 2, 128, 16
    g = gen(40)
    prompts, steps = [37, 1, 300], 20
    final = [n + steps for n in prompts]
    table, pool = table_for(final, page, g)
    kc, vc = (torch.full((pool, hkv, page, d), math.nan, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    cache = PagedKv(kc, vc, table)
    sin, cos = tables(max(final), d, 5)
    rope = Rope(sin, cos, 0)
    rows = normal(g, sum(prompts), hq + 2 * hkv, d)
    k_rot = torch.empty(sum(prompts), hkv, d, dtype=torch.bfloat16, device="cuda")
    lens, cu = ints(prompts), offsets(prompts)
    v = rows[:, hq + hkv:]
    q = gpu_ctx.kv_append(cache, rows[:, hq:hq + hkv], v, lens, cu, rope, q=rows[:, :hq], k_out=k_rot)
    out = gpu_ctx.attention_varlen(q, k_rot, v, cu)
    gpu_ctx.sync()
    packed_check(out, q, k_rot, v, prompts, prompts, True, "bf16")
    for s, n in enumerate(prompts):  # the cache holds what the prompt attention read
        ck, cv = gathered(cache, s, n)
        at = sum(prompts[:s])
        assert torch.equal(ck, k_rot[at:at + n]) and torch.equal(cv, v[at:at + n])
    # A single token's attention is the last row of the prompt's.
    last = gpu_ctx.attention_paged(q[(cu[1:] - 1).long()], cache, lens)
    paged_check(last, q[(cu[1:] - 1).long()], cache, prompts, "bf16")

    # Twenty steps as a captured graph whose lengths move on the device, against eager calls.
    steps_rows = normal(g, steps, 3, hq + 2 * hkv, d)
    eager = []
    twin = PagedKv(kc.clone(), vc.clone(), table)
    ws, l2 = gpu_ctx.paged_workspace(), lens.clone()
    for i in range(steps):
        l2 += 1
        r = steps_rows[i]
        qi = gpu_ctx.kv_append(twin, r[:, hq:hq + hkv], r[:, hq + hkv:], l2, rope=rope, q=r[:, :hq])
        eager.append(gpu_ctx.attention_paged(qi, twin, l2, workspace=ws))
        paged_check(eager[-1], qi, twin, [n + i + 1 for n in prompts], "bf16")
    token = steps_rows[0].clone()
    l3, ws3 = lens.clone(), gpu_ctx.paged_workspace()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        l3 += 1
        qi = gpu_ctx.kv_append(cache, token[:, hq:hq + hkv], token[:, hq + hkv:], l3, rope=rope, q=token[:, :hq])
        res = gpu_ctx.attention_paged(qi, cache, l3, workspace=ws3)
    for i in range(steps):
        token.copy_(steps_rows[i])
        graph.replay()
        assert torch.equal(res, eager[i])
    gpu_ctx.sync()
    for s, n in enumerate(final):
        for a, b in zip(gathered(cache, s, n), gathered(twin, s, n)):
            assert torch.equal(a, b)


def test_two_graphs_at_once(gpu_ctx):
    """Two captured steps with their own workspaces, replayed side by side on two streams."""
    g = gen(41)
    parts = []
    for i in range(2):
        lens = [4000 + 17 * i, 30, 900]
        q, cache = paged_case(g, 8, 2, 128, 16, lens, "bf16")
        n = [500, 31 + i]
        pq, pk, pv = normal(g, sum(n), 8, 128), normal(g, sum(n), 2, 128), normal(g, sum(n), 2, 128)
        cu, ls, ws = offsets(n), ints(lens), gpu_ctx.paged_workspace()
        want = (gpu_ctx.attention_paged(q, cache, ls), gpu_ctx.attention_varlen(pq, pk, pv, cu))
        graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            got = (gpu_ctx.attention_paged(q, cache, ls, workspace=ws), gpu_ctx.attention_varlen(pq, pk, pv, cu))
        parts.append((graph, stream, got, want, (q, cache, ls, pq, pk, pv, cu, ws)))
    for _ in range(20):
        for graph, stream, *_ in parts:
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for _, _, got, want, _ in parts:
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    gpu_ctx.sync()


def test_other_stream_and_second_context(gpu_ctx):
    g = gen(42)
    lens = [700, 90]
    q, cache = paged_case(g, 4, 4, 64, 16, lens, "f16")
    want = gpu_ctx.attention_paged(q, cache, ints(lens))
    gpu_ctx.sync()
    other, stream = GpuContext(0), torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = other.attention_paged(q, cache, ints(lens))
        other.sync()
    assert torch.equal(got, want)
    other.close()


def test_empty_calls(gpu_ctx):
    q, cache = paged_case(gen(43), 4, 2, 64, 16, [5], "bf16")
    none = torch.empty(0, 1, dtype=torch.int32, device="cuda")
    empty = PagedKv(cache.k, cache.v, none)
    assert gpu_ctx.attention_paged(q[:0], empty, ints([])).shape == (0, 4, 64)
    assert gpu_ctx.attention_varlen(q[:0], q[:0, :2], q[:0, :2], ints([0])).shape == (0, 4, 64)
    assert gpu_ctx.attention_varlen(q[:0], q[:0, :2], q[:0, :2], ints([0, 0, 0])).shape == (0, 4, 64)
    assert gpu_ctx.kv_append(empty, q[:0, :2], q[:0, :2], ints([])) is None
    out = torch.full_like(q, 4)
    gpu_ctx.attention_varlen(q, q[:, :2].contiguous(), q[:, :2].contiguous(), ints([0, 0]), out=out)  # all padding
    gpu_ctx.sync()
    assert (out == 4).all()
