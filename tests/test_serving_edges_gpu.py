"""The serving operators on the GPU at the places where their results, reports and promises are
easy to miss: offsets that do not fit the packed rows, keys that are not numbers at every position of
a tile, scores of any size, equal bits whatever the block table's width, a workspace that is ready
for the next call, refusals by the library itself.  Tolerances as in test_serving_gpu.py."""
from __future__ import annotations

import math

import pytest
import torch

from headshot_b200._lib import HS_ERR_INVALID, HS_ERR_TIMEOUT, HsError
from headshot_b200.engine import GpuContext, PagedKv, Rope
from test_serving_gpu import check_attention, gathered, gen, ints, normal, offsets, paged_case, paged_check, tables

pytestmark = pytest.mark.gpu


def reported(ctx, word):
    with pytest.raises(HsError) as e:
        ctx.sync()
    assert e.value.status == HS_ERR_INVALID and word in e.value.message


# -------------------------------------------------------------- kv_append --


@pytest.mark.parametrize("cu,healthy", [
    ([0, 20, 60], [0]),          # an end past the packed rows
    ([0, 30, 20], []),           # falling
    ([0, -5, 40], []),           # negative
    ([5, 20, 40], None),         # does not start at 0: tokens 0 to 4 belong to nobody
    ([0, 0, 2 ** 31 - 1], []),
    ([0, 10, 41], [0]),          # one past
    ([0, 40, 35], []),
])
def test_append_reports_bad_offsets_and_keeps_the_history(gpu_ctx, cu, healthy):
    """Offsets that do not rise from 0 within the rows are reported; a sequence whose end is wrong
    appends nothing, so its history keeps its rows, and a healthy one gets exactly its tokens."""
    g = gen(len(cu) + cu[1])
    lens = [40, 100]  # rows after the append, histories before it
    _, cache = paged_case(g, 4, 2, 64, 16, lens, "bf16")
    k0, v0 = cache.k.clone(), cache.v.clone()
    k, v, q = normal(g, 40, 2, 64), normal(g, 40, 2, 64), normal(g, 40, 4, 64)
    gpu_ctx.kv_append(cache, k, v, ints(lens), cu_new=ints(cu), q=q)
    reported(gpu_ctx, "offsets")
    if healthy is not None:
        for s in healthy:
            p = torch.arange(lens[s] - (cu[s + 1] - cu[s]), lens[s], device="cuda")
            at, off = cache.block_table[s][p // 16].long(), p % 16
            k0[at, :, off], v0[at, :, off] = k[cu[s]:cu[s + 1]], v[cu[s]:cu[s + 1]]
        assert torch.equal(cache.k, k0) and torch.equal(cache.v, v0)
    gpu_ctx.kv_append(cache, k, v, ints(lens), cu_new=ints([0, 20, 40]))
    gpu_ctx.sync()  # the context goes on
    for s in range(2):
        ck, cv = gathered(cache, s, lens[s])
        assert torch.equal(ck[-20:], k[20 * s:20 * s + 20]) and torch.equal(cv[-20:], v[20 * s:20 * s + 20])


def test_append_reports_one_falling_pair_among_many_sequences(gpu_ctx):
    """A pair that no token's own sequence shows, first, last and far from both."""
    n_seqs = 5000
    table = torch.arange(n_seqs, device="cuda", dtype=torch.int32)[:, None].contiguous()
    kc, vc = (torch.zeros(n_seqs, 1, 4, 64, dtype=torch.float16, device="cuda") for _ in range(2))
    g = gen(2)
    for tokens in (1, 700):
        k, v = normal(g, tokens, 1, 64, dtype="f16"), normal(g, tokens, 1, 64, dtype="f16")
        cu = torch.zeros(n_seqs + 1, dtype=torch.int32, device="cuda")
        cu[n_seqs // 2:] = tokens
        lens = torch.full((n_seqs,), 4, dtype=torch.int32, device="cuda")
        for at in (1, n_seqs // 4, n_seqs // 2 - 1):  # a rise and a fall among empty sequences
            bad = cu.clone()
            bad[at] = 1 if tokens == 1 else 3
            bad[n_seqs // 2:] = tokens
            if at + 1 == n_seqs // 2:
                bad[at] = tokens + 5
            gpu_ctx.kv_append(PagedKv(kc, vc, table), k, v, lens, cu_new=bad)
            reported(gpu_ctx, "offsets")
        # the pad rows behind the last sequence are no fault
        cu[n_seqs // 2:] = tokens // 2
        gpu_ctx.kv_append(PagedKv(kc, vc, table), k, v, lens, cu_new=cu)
        gpu_ctx.sync()


def test_append_bad_page_leaves_the_rest_exact(gpu_ctx):
    """One sequence's bad page, length or rotation row: the others' tokens are written exactly, and
    nothing else of either cache changes."""
    g = gen(24)
    k, v = normal(g, 3, 2, 64), normal(g, 3, 2, 64)
    _, cache = paged_case(g, 4, 2, 64, 16, [40, 40, 40], "bf16")
    for what, lens, rope, word in (("page", [40, 40, 40], None, "page"), ("length", [40, 49, 40], None, "length"),
                                   # rows below the prefix of 30 pass through; position 39 asks for row 9 of 9
                                   ("row", [30, 40, 30], Rope(*tables(9, 64, 2), 30), "rotation")):
        kc, vc, table = cache.k.clone(), cache.v.clone(), cache.block_table.clone()
        if what == "page":
            table[1, 2] = kc.shape[0]
        want_k, want_v = kc.clone(), vc.clone()
        for s in (0, 2):
            p = lens[s] - 1
            at = table[s, p // 16].long()
            want_k[at, :, p % 16], want_v[at, :, p % 16] = k[s], v[s]
        gpu_ctx.kv_append(PagedKv(kc, vc, table), k, v, ints(lens), rope=rope)
        reported(gpu_ctx, word)
        assert torch.equal(kc, want_k) and torch.equal(vc, want_v)


# --------------------------------------------------------------- NaN keys --


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("d", [64, 128])
def test_one_nan_key_reaches_every_row_that_sees_it(gpu_ctx, dtype, d):
    """A NaN score makes its row NaN, whichever position of a key tile it has, and no other row."""
    g = gen(d)
    n = 200  # two and more tiles of 64 and 96 keys: every position of a first and of a later tile
    q = normal(g, n, 2, d, dtype=dtype)  # sequence p: one query, n keys, key p is not a number
    k, v = normal(g, n, n, 1, d, dtype=dtype), normal(g, n * n, 1, d, dtype=dtype)
    p = torch.arange(n, device="cuda")
    k[p, p, 0, p % d] = math.nan
    out = gpu_ctx.attention_varlen(q, k.view(n * n, 1, d), v, offsets([1] * n), cu_k=offsets([n] * n), causal=False)
    gpu_ctx.sync()
    assert out.isnan().all()

    kc = normal(g, n, 1, d, dtype=dtype)
    clean = gpu_ctx.attention_varlen(q, kc, v[:n], offsets([n]))
    for at in (0, 63, 64, 95, 96, 127, 150, 191, 192, 199):
        kn = kc.clone()
        kn[at, 0, 3] = math.nan
        out = gpu_ctx.attention_varlen(q, kn, v[:n], offsets([n]))
        gpu_ctx.sync()
        assert out[at:].isnan().all() and torch.equal(out[:at], clean[:at])


@pytest.mark.parametrize("d", [64, 128])
def test_one_nan_key_in_the_cache(gpu_ctx, d):
    n = 150
    g = gen(d + 1)
    q, cache = paged_case(g, 4, 2, d, 16, [n] * n, "bf16")
    p = torch.arange(n, device="cuda")
    cache.k[cache.block_table[p, p // 16].long(), 0, p % 16, 5] = math.nan  # key p of sequence p, first key head
    out = gpu_ctx.attention_paged(q, cache, ints([n] * n))
    gpu_ctx.sync()
    assert out[:, :2].isnan().all() and torch.isfinite(out[:, 2:]).all()


# ------------------------------------------------------------ packed rows --


@pytest.mark.parametrize("causal", [True, False])
def test_offsets_into_a_larger_pack(gpu_ctx, causal):
    """A slice of a pack's offsets attends for its sequences alone; rows before and behind stay."""
    g = gen(31)
    lens = [30, 130, 1, 70, 9]
    q, k, v = normal(g, 240, 4, 64), normal(g, 240, 2, 64), normal(g, 240, 2, 64)
    cu = offsets(lens)
    whole = gpu_ctx.attention_varlen(q, k, v, cu, causal=causal)
    out = torch.full_like(q, 7)
    gpu_ctx.attention_varlen(q, k, v, cu[1:4].contiguous(), causal=causal, out=out)
    gpu_ctx.sync()
    assert (out[:30] == 7).all() and torch.equal(out[30:161], whole[30:161]) and (out[161:] == 7).all()


# ------------------------------------------------------------ score range --


@pytest.mark.parametrize("dtype,size", [("bf16", 2e3), ("bf16", 1e5), ("bf16", 1e9), ("bf16", 1e15), ("f16", 2e3), ("f16", 6e4)])
@pytest.mark.parametrize("d", [64, 128])
def test_prompt_scores_of_any_size(gpu_ctx, dtype, size, d):
    """Each row belongs to its largest score, which the inputs set apart from the others by far: score
    d size^2, the next one 2 size^2 less at least."""
    g = gen(18)
    n = 130
    sign = torch.where(torch.rand(n, 1, d, generator=g, device="cuda") < 0.5, -1.0, 1.0)
    k = (sign * size).to(torch.bfloat16 if dtype == "bf16" else torch.float16)
    q = k.flip(0)
    v = normal(g, n, 1, d, dtype=dtype)
    out = gpu_ctx.attention_varlen(q, k, v, offsets([n]), causal=False)
    gpu_ctx.sync()
    check_attention(out, v.flip(0).double(), v.flip(0).double().abs(), n, dtype, v.abs().max().item())


@pytest.mark.parametrize("dtype,size", [("bf16", 1.0), ("bf16", 2.0 ** 10), ("bf16", 2.0 ** 20), ("bf16", 2.0 ** 60), ("f16", 2.0 ** 10), ("f16", 2.0 ** 15)])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("step", [1, -1])
def test_prompt_maximum_that_moves_through_every_size(gpu_ctx, dtype, size, d, step):
    """Key j scores d size (j - 150) before the scale, rising or falling: with at least d / sqrt(d) = 8
    between neighbours a row is its largest key's value but for weights of e^-8 and less, which the
    reference counts; sizes run from small scores to ones whose spacing in f32 is many binades."""
    g = gen(19)
    n = 300
    t = torch.bfloat16 if dtype == "bf16" else torch.float16
    j = torch.arange(n, device="cuda") - 150
    j = torch.where(j.abs() > 128, j.sign() * 128, j)  # whole in bf16 too; ties at both ends share their weight
    k = (j * step).to(t)[:, None, None].expand(n, 1, d).contiguous()
    q = torch.full((n, 2, d), size, dtype=t, device="cuda")
    v = normal(g, n, 1, d, dtype=dtype)
    out = gpu_ctx.attention_varlen(q, k, v, offsets([n]))
    gpu_ctx.sync()
    # every product and partial sum is whole times size, so scores are exact in f32 and in f64
    s = torch.outer(torch.ones(n, device="cuda", dtype=torch.float64), j.double() * step) * (d * size * d ** -0.5)
    s = s.masked_fill(torch.ones_like(s, dtype=torch.bool).triu(1), -math.inf)
    w = torch.softmax(s, -1)
    ref, mass = w @ v[:, 0].double(), w @ v[:, 0].double().abs()
    for h in range(2):
        check_attention(out[:, h], ref, mass, n, dtype, v.abs().max().item())


# -------------------------------------------------------------- time-outs --


@pytest.mark.parametrize("d", [64, 128])
def test_prompt_gives_up_while_it_rescales(d):
    """Wait bound 0 on scores whose maximum moves with every tile: a row that waits to rescale its
    output gives up too, and the next call with the usual bound is right."""
    ctx = GpuContext(0)
    g = gen(60)
    n = 1500
    q = torch.full((n, 4, d), 2.0, dtype=torch.bfloat16, device="cuda")
    k = (torch.arange(n, device="cuda") / 8).to(torch.bfloat16)[:, None, None].expand(n, 2, d).contiguous()
    v = normal(g, n, 2, d)
    good = ctx.attention_varlen(q, k, v, offsets([n]))
    ctx.sync()
    for _ in range(5):
        ctx.set_wait_timeout_ms(0)
        ctx.attention_varlen(q, k, v, offsets([n]))
        with pytest.raises(HsError) as e:
            ctx.sync()
        assert e.value.status == HS_ERR_TIMEOUT
        ctx.set_wait_timeout_ms(2000)
        again = ctx.attention_varlen(q, k, v, offsets([n]))
        ctx.sync()
        assert torch.equal(good, again)
    ctx.close()


# ------------------------------------------------------------ paged split --


@pytest.mark.parametrize("hq,hkv,d", [(32, 8, 128), (16, 16, 64), (4, 1, 128)])
@pytest.mark.parametrize("lens", [[8191], [5000, 17, 700, 0, 2300]])
def test_paged_bits_do_not_depend_on_the_table_width(gpu_ctx, hq, hkv, d, lens):
    """The split of the keys over the GPU follows the lengths, not the room that the table has."""
    q, cache = paged_case(gen(50), hq, hkv, d, 16, lens, "bf16")
    outs = []
    for wide in (0, 3, 700, 20000):
        table = torch.full((len(lens), cache.block_table.shape[1] + wide), -1, dtype=torch.int32, device="cuda")
        table[:, :cache.block_table.shape[1]] = cache.block_table
        outs.append(gpu_ctx.attention_paged(q, PagedKv(cache.k, cache.v, table), ints(lens)))
    gpu_ctx.sync()
    for x in outs[1:]:
        assert torch.equal(outs[0], x)
    paged_check(outs[0], q, cache, lens, "bf16")


def test_paged_leaves_its_workspace_ready(gpu_ctx):
    """The counters (the first 4 KiB) are zero again after every call, so the next one may be of any shape."""
    ws = gpu_ctx.paged_workspace()
    for seqs, longest, hq, hkv, d in ((1, 30000, 8, 8, 128), (300, 40, 4, 2, 64), (37, 3001, 8, 8, 64), (2, 20001, 48, 1, 128),
                                      (700, 9, 2, 1, 128), (1, 9000, 2, 1, 64)):
        g = gen(seqs)
        lens = torch.randint(0, longest + 1, (seqs,), generator=g, device="cuda").tolist()
        lens[-1] = longest
        q, cache = paged_case(g, hq, hkv, d, 16, lens, "bf16")
        outs = []
        for _ in range(2):
            outs.append(gpu_ctx.attention_paged(q, cache, ints(lens), workspace=ws))
            gpu_ctx.sync()
            assert (ws[:4096] == 0).all()
        assert torch.equal(*outs)
        paged_check(outs[0], q, cache, lens, "bf16")
    assert (ws[4096:] != 0).any()  # the calls did cut sequences


# --------------------------------------------------------------- refusals --


def test_the_library_refuses_by_itself(gpu_ctx):
    """Through the C ABI, past the Python checks: each call returns a status and launches nothing."""
    L, h = gpu_ctx._L, gpu_ctx._h
    x = torch.zeros(1 << 16, dtype=torch.bfloat16, device="cuda")
    i = torch.zeros(64, dtype=torch.int32, device="cuda")
    f = torch.zeros(1 << 12, dtype=torch.float32, device="cuda")
    ws = gpu_ctx.paged_workspace()
    X, I, F, bf16 = x.data_ptr(), i.data_ptr(), f.data_ptr(), 2

    def append(q=X, k=X, v=X, qo=X + 32768, ko=0, kc=X, vc=X, table=I, lens=I, cu=0, qs=0, ks=0, vs=0, n=2, seqs=2, hq=4,
               hkv=2, d=64, pages=4, page=16, most=2, dt=bf16, sin=0, cos=0, rows=0, prefix=0, tpf=0):
        return L.hs_kv_append(h, q, k, v, qo, ko, kc, vc, table, lens, cu, qs, ks, vs, n, seqs, hq, hkv, d, pages, page, most,
                              dt, sin, cos, rows, prefix, tpf)

    def varlen(q=X, k=X, v=X, out=X, qs=0, ks=0, vs=0, cq=I, ck=0, tq=2, tk=2, seqs=1, hq=4, hkv=2, d=64, causal=1, dt=bf16):
        return L.hs_attention_varlen(h, q, k, v, out, qs, ks, vs, cq, ck, tq, tk, seqs, hq, hkv, d, causal, dt, 0.0)

    def paged(q=X, out=X, kc=X, vc=X, table=I, lens=I, qs=0, seqs=2, hq=4, hkv=2, d=64, pages=4, page=16, most=2, dt=bf16,
              w=ws.data_ptr(), nb=ws.nbytes):
        return L.hs_attention_paged(h, q, out, kc, vc, table, lens, qs, seqs, hq, hkv, d, pages, page, most, dt, 0.0, w, nb)

    bad = [
        *(append(**{a: 0}) for a in ("k", "v", "qo", "kc", "vc", "table", "lens", "hkv", "page", "q")),
        *(append(**{a: X + 2}) for a in ("q", "k", "v", "qo", "ko", "kc", "vc")), append(table=I + 2), append(cu=I + 1),
        append(n=3), append(hq=5), append(hq=1026), append(hq=4096, hkv=2048), append(d=96), append(dt=0), append(dt=9),
        append(qs=100), append(ks=129), append(vs=64), append(sin=F), append(sin=F, cos=F + 4), append(pages=2 ** 31),
        append(page=2 ** 16, most=2 ** 16), append(sin=F, cos=F, rows=18, prefix=5, tpf=24),
        append(sin=F, cos=F, rows=18, prefix=25, tpf=24), append(qo=X, qs=512), append(ko=X, ks=256),
        append(n=2 ** 31, cu=I), append(seqs=2 ** 31 - 1, cu=I),
        *(varlen(**{a: 0}) for a in ("q", "k", "v", "out", "cq", "hkv")), *(varlen(**{a: X + 8}) for a in ("q", "k", "v", "out")),
        varlen(cq=I + 2), varlen(tk=3), varlen(hq=129 * 2), varlen(hq=3), varlen(d=32), varlen(dt=0), varlen(qs=250),
        varlen(ks=64), varlen(vs=132), varlen(tq=2 ** 31, tk=2 ** 31), varlen(seqs=2 ** 31 - 1),
        varlen(qs=2 ** 33),
        *(paged(**{a: 0}) for a in ("q", "out", "kc", "vc", "table", "lens", "hkv", "page", "w")),
        *(paged(**{a: X + 8}) for a in ("q", "out", "kc", "vc")), paged(w=ws.data_ptr() + 8), paged(nb=ws.nbytes - 1),
        paged(hq=3), paged(d=96), paged(dt=0), paged(qs=8), paged(seqs=2 ** 30), paged(pages=2 ** 32 - 1),
    ]
    assert all(s != 0 for s in bad), [n for n, s in enumerate(bad) if s == 0]
    gpu_ctx.sync()


def test_outputs_in_place_and_overlapping(gpu_ctx):
    """The queries' own contiguous rows may take the output; any other overlap with an input is refused."""
    g = gen(70)
    lens = [300, 45, 1, 129]
    n = sum(lens)
    for hq, hkv, d in ((4, 4, 64), (6, 2, 128), (10, 2, 64)):
        q, k, v = normal(g, n, hq, d), normal(g, n, hkv, d), normal(g, n, hkv, d)
        for causal in (True, False):
            want = gpu_ctx.attention_varlen(q, k, v, offsets(lens), causal=causal)
            here = q.clone()
            assert gpu_ctx.attention_varlen(here, k, v, offsets(lens), causal=causal, out=here) is here
            gpu_ctx.sync()
            assert torch.equal(here, want)
        klens = [3000, 45, 0, 129]
        pq, cache = paged_case(g, hq, hkv, d, 16, klens, "bf16")
        want = gpu_ctx.attention_paged(pq, cache, ints(klens))
        assert gpu_ctx.attention_paged(pq, cache, ints(klens), out=pq) is pq
        gpu_ctx.sync()
        assert torch.equal(pq, want)
    q, k, v = normal(g, n, 4, 64), normal(g, n, 4, 64), normal(g, n, 4, 64)
    buf = normal(g, 2 * n, 4, 64)
    _, cache = paged_case(g, 4, 4, 64, 16, [20, 20], "bf16")
    fused = normal(g, 2, 12, 64)
    lens2 = ints([20, 20])
    for call in (lambda: gpu_ctx.attention_varlen(q, k, v, offsets(lens), out=k),
                 lambda: gpu_ctx.attention_varlen(q, k, v, offsets(lens), out=v),
                 lambda: gpu_ctx.attention_varlen(buf[:n], k, v, offsets(lens), out=buf[5:n + 5]),
                 lambda: gpu_ctx.attention_varlen(q, buf[:n], v, offsets(lens), out=buf[n - 1:2 * n - 1]),
                 lambda: gpu_ctx.attention_paged(buf[1:3], cache, lens2, out=buf[0:2]),
                 lambda: gpu_ctx.kv_append(cache, k[:2], v[:2], lens2, q=q[:2], q_out=k[:2]),
                 lambda: gpu_ctx.kv_append(cache, k[:2], v[:2], lens2, k_out=v[:2]),
                 lambda: gpu_ctx.kv_append(cache, k[:2], v[:2], lens2, q=q[:2], q_out=buf[:2], k_out=buf[1:3]),
                 lambda: gpu_ctx.kv_append(cache, k[:2], v[:2], lens2, q=q[:2], k_out=q[:2]),
                 lambda: gpu_ctx.kv_append(cache, k[:2], v[:2], lens2, k_out=k[1:3]),
                 lambda: gpu_ctx.kv_append(cache, fused[:, 4:8], fused[:, 8:], lens2, q=fused[:, :4],
                                           q_out=fused.view(-1, 4, 64)[:2])):
        with pytest.raises(HsError) as e:
            call()
        assert e.value.status == HS_ERR_INVALID
    gpu_ctx.sync()
    gpu_ctx.attention_varlen(buf[:n], k, v, offsets(lens), out=buf[n:])  # side by side in one buffer
    gpu_ctx.kv_append(cache, fused[:, 4:8], fused[:, 8:], lens2, q=fused[:, :4], q_out=buf[:2], k_out=buf[2:4])
    gpu_ctx.sync()
