"""Windowed attention with sinks, packed and against a cache, compared with
64-bit softmax attention under an explicit mask, and its refusals."""
import ctypes

import pytest
import torch

from h3_engine_b200 import _lib, ops

BF16, F16 = torch.bfloat16, torch.float16


def seen_mask(n_q, n_k, left, right, sinks, causal):
    p = torch.arange(n_q)[:, None] + (n_k - n_q)
    j = torch.arange(n_k)[None, :]
    left = 10 ** 9 if left is None else left
    right = 10 ** 9 if right is None else right
    see = ((j >= p - left) & (j <= p + right)) | (j < sinks)
    return see & (j <= p) if causal else see


def attend(q, k, v, see, scale, half):
    """(64-bit attention of [n_q, D] x [n_k, D], bound on the kernel's error).

    The kernel's logits are fp32 sums of exact products: off by at most
    D * 2^-23 * sum |q k| * scale.  exp2 and its polynomial are off by 1.2e-4
    relative at most, P is rounded to 16 bits (``half`` relative), the
    accumulations by 2^-23 per key.  A relative error r of every weight moves a
    weighted mean by at most 2 r * sum p |v|; then the output's own rounding."""
    q, k, v = q.double(), k.double(), v.double()
    if not k.shape[0]:
        z = torch.zeros_like(q)
        return z, z
    z = (q @ k.T) * scale
    dz = (q.abs() @ k.abs().T).amax(-1, keepdim=True) * scale * q.shape[1] * 2.0 ** -23
    p = torch.softmax(z.masked_fill(~see, -1e300), -1) * see
    o = p @ v
    r = dz + 1.3e-4 + half + k.shape[0] * 2.0 ** -23
    off = 2 * r * (p @ v.abs())
    return o, off + half * (o.abs() + off)


def check(got, want, off):
    assert torch.isfinite(got).all()
    assert ((got.double() - want).abs() <= off + 1e-7).all(), \
        float(((got.double() - want).abs() - off).max())


def packed_case(lens_q, lens_k, heads, kv, d, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    rq, rk = sum(lens_q), sum(lens_k)
    q = (torch.randn(rq, heads * d, generator=g) * 1.5).to(dtype)
    k = torch.randn(rk, kv * d, generator=g).to(dtype)
    v = torch.randn(rk, kv * d, generator=g).to(dtype)
    cq = [0] + torch.tensor(lens_q).cumsum(0).tolist()
    ck = [0] + torch.tensor(lens_k).cumsum(0).tolist()
    return q, k, v, cq, ck


def check_packed(got, q, k, v, cq, ck, heads, kv, d, rule):
    half = torch.finfo(q.dtype).eps / 2
    for a, b, s, e in zip(cq[:-1], cq[1:], ck[:-1], ck[1:]):
        if a == b:
            continue
        see = seen_mask(b - a, e - s, *rule)
        for h in range(heads):
            m = h // (heads // kv)
            want, off = attend(q[a:b, h * d:(h + 1) * d], k[s:e, m * d:(m + 1) * d],
                               v[s:e, m * d:(m + 1) * d], see, d ** -0.5, half)
            check(got[a:b, h * d:(h + 1) * d], want, off)
            assert (got[a:b, h * d:(h + 1) * d][~see.any(-1)] == 0).all()


# ---------------------------------------------------------------- CPU: refusals
def test_host_checks_refuse_without_a_gpu():
    lib = _lib.lib()
    p, odd = ctypes.c_void_p(1 << 20), ctypes.c_void_p((1 << 20) + 4)

    def packed(q=p, stride=256, dtype=0, H=2, kv=1, D=128, qs=(0,), ql=(4,), ks=(0,), kl=(4,),
               rows=8, left=0, right=0, sinks=0, causal=0, scale=0.1, out=p):
        arr = [(ctypes.c_int32 * len(t))(*t) for t in (qs, ql, ks, kl)]
        return lib.h3b_attention_window(q, rows, stride, p, 128, p, 128, rows, dtype, H, kv, D,
                                        *arr, len(qs), left, right, sinks, causal, scale, out,
                                        256, None, 0, None)

    assert packed(D=96) == 1 and packed(dtype=2) == 1 and packed(H=3, kv=2) == 1
    assert packed(H=0) == 1 and packed(scale=0.0) == 1 and packed(scale=float("nan")) == 1
    assert packed(left=-1) == 1 and packed(right=-1) == 1 and packed(sinks=-1) == 1
    assert packed(causal=2) == 1 and packed(stride=128) == 1 and packed(stride=260) == 2
    assert packed(qs=(5,)) == 1 and packed(ks=(5,)) == 1 and packed(ql=(-1,)) == 1
    assert packed(kl=(9,)) == 1 and packed(qs=(-1,)) == 1
    assert packed(q=odd) == 2 and packed(q=None) == 1 and packed(out=None) == 1
    assert packed(ql=(0,)) == 0

    def decode(q=p, k=p, length=p, B=2, room=64, n=1, dtype=0, H=4, kv=2, D=128, left=0, scale=0.1,
               qst=(512, 512, 128)):
        st = [(ctypes.c_int64 * 3)(*t) for t in (qst, (16384, 256, 128), (16384, 256, 128))]
        return lib.h3b_attention_window_decode(q, st[0], k, st[1], p, st[2], length, B, room, n,
                                               dtype, H, kv, D, left, 0, 0, 1, scale, p, None)

    assert decode(D=32) == 1 and decode(dtype=2) == 1 and decode(H=3) == 1 and decode(B=-1) == 1
    assert decode(left=-1) == 1 and decode(scale=-1.0) == 1 and decode(room=1 << 31) == 1
    assert decode(qst=(512, 512, 129)) == 2 and decode(qst=(-512, 512, 128)) == 1
    assert decode(q=odd) == 2 and decode(length=None) == 1 and decode(k=None) == 1
    assert decode(B=0) == 0 and decode(n=0) == 0


def test_scale_must_be_finite_and_workspace_sizes_hold_for_huge_rules():
    lib = _lib.lib()
    p = ctypes.c_void_p(1 << 20)
    one, zero, huge = (ctypes.c_int32 * 1)(4), (ctypes.c_int32 * 1)(0), (1 << 63) - 1
    assert lib.h3b_attention_window(p, 4, 128, p, 128, p, 128, 4, 0, 1, 1, 128, zero, one, zero,
                                    one, 1, 0, 0, 0, 0, float("inf"), p, 128, None, 0, None) == 1
    long = (ctypes.c_int32 * 1)(4000)
    need = lib.h3b_attention_window_ws(long, long, 1, 2, 128, 4000, 4000, 0)
    assert need > 0
    for left, right, sinks in ((huge, huge, huge), (huge, 0, 0), (0, 0, huge)):
        assert lib.h3b_attention_window_ws(long, long, 1, 2, 128, left, right, sinks) == need


def test_cpu_tensors_are_refused():
    x = torch.zeros(4, 128, dtype=BF16)
    with pytest.raises(ValueError):
        ops.attention_window(x, x, x, 1, 128, [0, 4])
    c = torch.zeros(1, 4, 1, 128, dtype=BF16)
    with pytest.raises(ValueError):
        ops.attention_window_decode(c, c, c, torch.zeros(1, dtype=torch.int32))


@pytest.mark.parametrize("name", ["attention_window", "attention_window_decode"])
def test_operators_declare_their_outputs(name):
    schema = getattr(torch.ops.h3b, name + "_out").default._schema
    assert {a.name for a in schema.arguments
            if a.alias_info is not None and a.alias_info.is_write} == {"out"}


def test_operators_trace_without_a_gpu():
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        q = torch.empty(10, 256, dtype=BF16, device="cuda")
        assert ops.attention_window(q, q, q, 2, 128, [0, 10]).shape == (10, 256)
        c = torch.empty(2, 8, 2, 64, dtype=BF16, device="cuda")
        n = torch.empty(2, dtype=torch.int32, device="cuda")
        assert ops.attention_window_decode(c[:, :1], c, c, n).shape == (2, 1, 2, 64)


# ---------------------------------------------------------------- GPU: packed
RULES = [(None, None, 0, False), (None, None, 0, True), (0, 0, 0, False), (0, 0, 3, True),
         (63, 17, 0, False), (127, 128, 5, False), (200, 0, 130, True), (1000, 40, 300, False),
         (5, None, 0, True), (None, 5, 2, False)]


@pytest.mark.gpu
@pytest.mark.parametrize("rule", RULES)
@pytest.mark.parametrize("d,dtype", [(128, BF16), (64, F16)])
def test_packed_documents(cuda, rule, d, dtype):
    lens = [1, 300, 0, 128, 129, 257, 7, 640]
    q, k, v, cq, ck = packed_case(lens, lens, 2, 1, d, dtype)
    got = ops.attention_window(q.to(cuda), k.to(cuda), v.to(cuda), 2, d, cq, kv_heads=1,
                               window=rule[:2], sinks=rule[2], causal=rule[3])
    check_packed(got.cpu(), q, k, v, cq, ck, 2, 1, d, rule)


@pytest.mark.gpu
@pytest.mark.parametrize("rule", [(None, None, 0, True), (100, 0, 4, True), (30, 500, 0, False)])
@pytest.mark.parametrize("d,dtype", [(128, F16), (64, BF16)])
def test_queries_and_keys_of_different_lengths(cuda, rule, d, dtype):
    """Chunks of new queries against longer histories, documents with more
    queries than keys (their first queries may see nothing) and without keys."""
    lq, lk = [1, 64, 200, 300, 40, 5], [500, 700, 200, 100, 0, 129]
    q, k, v, cq, ck = packed_case(lq, lk, 4, 2, d, dtype, seed=1)
    got = ops.attention_window(q.to(cuda), k.to(cuda), v.to(cuda), 4, d, cq, kv_heads=2,
                               cu_seqlens_k=ck, window=rule[:2], sinks=rule[2], causal=rule[3])
    check_packed(got.cpu(), q, k, v, cq, ck, 4, 2, d, rule)


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,heads,kv,d", [
    (1500, 2, 1, 128),      # items of 128 queries, their keys in parts
    (2200, 2, 2, 64),       # the same, head_dim 64
    (2100, 8, 4, 128),      # items of 256 in parts
    (2100, 8, 8, 64),       # the same in steps of 128 keys
    (1300, 52, 13, 64),     # whole waves of steps of 64 keys, the rest in parts
])
@pytest.mark.parametrize("rule", [(None, None, 0, False), (700, 500, 70, True)])
def test_items_and_parts(cuda, tokens, heads, kv, d, rule):
    q, k, v, cq, ck = packed_case([tokens], [tokens], heads, kv, d, BF16, seed=5)
    got = ops.attention_window(q.to(cuda), k.to(cuda), v.to(cuda), heads, d, cq, kv_heads=kv,
                               window=rule[:2], sinks=rule[2], causal=rule[3])
    check_packed(got.cpu(), q, k, v, cq, ck, heads, kv, d, rule)


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128])
def test_launches_that_share_their_counters(cuda, d):
    """More documents than one launch takes, each launch with keys in parts."""
    lq = [3 + i % 4 for i in range(70)]
    lk = [1100 + 3 * i for i in range(70)]
    q, k, v, cq, ck = packed_case(lq, lk, 1, 1, d, F16, seed=6)
    for rule in ((None, None, 0, True), (900, 0, 40, True)):
        got = ops.attention_window(q.to(cuda), k.to(cuda), v.to(cuda), 1, d, cq, cu_seqlens_k=ck,
                                   window=rule[:2], sinks=rule[2], causal=rule[3])
        check_packed(got.cpu(), q, k, v, cq, ck, 1, 1, d, rule)


@pytest.mark.gpu
def test_many_documents_and_large_logits(cuda):
    lens = [3 + i % 5 for i in range(150)]
    q, k, v, cq, ck = packed_case(lens, lens, 1, 1, 64, BF16, seed=2)
    rule = (2, 1, 1, False)
    q = q * 40
    got = ops.attention_window(q.to(cuda), k.to(cuda), v.to(cuda), 1, 64, cq, window=rule[:2],
                               sinks=rule[2])
    check_packed(got.cpu(), q, k, v, cq, ck, 1, 1, 64, rule)


def one_hot_rows(q, k, see, scale):
    """The key each query picks, and which queries pick one for certain: where the
    second logit is further below than the kernel's error on both and the
    exponent that rounds to 0, every weight but one is exactly 0."""
    q, k = q.double(), k.double()
    z = (q @ k.T * scale).masked_fill(~see, -1e300)
    dz = (q.abs() @ k.abs().T).amax(-1) * scale * (q.shape[1] + 2) * 2.0 ** -23
    top = z.topk(2, -1).values
    return z.argmax(-1), top[:, 0] - top[:, 1] > 2 * dz + 200


@pytest.mark.gpu
@pytest.mark.parametrize("size", [2.0 ** 10, 2.0 ** 14, 2.0 ** 30])
@pytest.mark.parametrize("d", [64, 128])
def test_huge_logits_pick_one_key(cuda, size, d):
    """Logits of 10^7 ... 10^18: one weight is 1 and the others 0."""
    n, rule = 300, (200, 50, 3, False)
    q, k, v, cq, _ = packed_case([n], [n], 2, 1, d, BF16, seed=8)
    q, k = q * size, k * size
    dev = [t.to(cuda) for t in (q, k, v)]
    got = ops.attention_window(*dev, 2, d, cq, kv_heads=1, window=rule[:2], sinks=rule[2]).cpu()
    one = ops.attention_window_decode(
        dev[0].view(1, n, 2, d), dev[1].view(1, n, 1, d), dev[2].view(1, n, 1, d),
        torch.tensor([n], dtype=torch.int32, device=cuda), window=rule[:2], sinks=rule[2],
        causal=False).cpu().view(n, 2 * d)
    see = seen_mask(n, n, *rule)
    for h in range(2):
        c = slice(h * d, h * d + d)
        pick, sure = one_hot_rows(q[:, c], k, see, d ** -0.5)
        assert sure.float().mean() > 0.5
        # out = round16(round16(P) v / P): P is 2^(z - m) for a maximum m so far, no
        # power of two, so its rounding shows beside the output's: half a step each
        # (their product and the division's 2^-22 are in the 1 %)
        for o in (got, one):
            assert ((o[sure, c].double() - v[pick[sure]].double()).abs()
                    <= 2.01 * 2.0 ** -8 * v[pick[sure]].double().abs()).all()
        assert torch.isfinite(got[:, c]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128])
def test_infinite_logits(cuda, d):
    """A visible key whose logit is -inf weighs nothing; a row that sees only such
    keys, or one whose logit is +inf or NaN, is NaN; a row that sees none is 0."""
    n = 40
    q, k, v, cq, _ = packed_case([n], [n], 1, 1, d, BF16, seed=9)
    q = q.abs() + 0.1
    inf = float("inf")
    k[5], k[20:24], k[30], k[35, 0] = -inf, -inf, inf, float("nan")
    left, right = 2, 0
    z = (q.double() @ k.double().T) * d ** -0.5
    see = seen_mask(n, n, left, right, 0, False)
    want = torch.softmax(z.masked_fill(~see, -inf), -1)
    dead = want.isnan().any(-1)
    assert dead.tolist() == [i in (22, 23, 30, 31, 32, 35, 36, 37) for i in range(n)]
    dev = [t.to(cuda) for t in (q, k, v)]
    got = ops.attention_window(*dev, 1, d, cq, window=(left, right)).cpu()
    one = ops.attention_window_decode(
        dev[0].view(1, n, 1, d), *(t.view(1, n, 1, d) for t in dev[1:]),
        torch.tensor([n], dtype=torch.int32, device=cuda), window=(left, right)).cpu().view(n, d)
    # attend()'s terms against max |v|: twice P's half step and the logits' 4e-4
    # (scaled sums |q k| of at most 16.1, times D 2^-23: 2.5e-4; exponentials 1.3e-4),
    # then the output's half step
    tol = (2 * (2.0 ** -8 + 4e-4) + 1.02 * 2.0 ** -8) * v.double().abs().amax()
    ref = (want.nan_to_num() @ v.double())[~dead]
    for o in (got, one):
        assert torch.isnan(o[dead]).all()
        assert ((o[~dead].double() - ref).abs() <= tol).all()


@pytest.mark.gpu
def test_equals_full_attention_without_a_window(cuda):
    q, k, v, cq, _ = packed_case([700, 333], [700, 333], 2, 2, 128, BF16)
    dev = [t.to(cuda) for t in (q, k, v)]
    a = ops.attention_window(*dev, 2, 128, cq).cpu().double()
    b = ops.attention_qkv(*dev, 2, 128, cq).cpu().double()
    # Both kernels round P to bf16 from exponentials that differ by up to 1.2e-4
    # (which keys take the polynomial, where the keys are split), so their
    # results differ by P's rounding steps against sum p |v|, not against |o|:
    # each is within attend()'s bound of the exact result, so they are within
    # twice that of each other.
    for s, e in zip(cq[:-1], cq[1:]):
        see = torch.ones(e - s, e - s, dtype=torch.bool)
        for h in (0, 1):
            c = slice(h * 128, h * 128 + 128)
            _, off = attend(q[s:e, c], k[s:e, c], v[s:e, c], see, 128 ** -0.5, 2.0 ** -8)
            assert ((a[s:e, c] - b[s:e, c]).abs() <= 2 * off).all()


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128])
def test_rows_nobody_sees_do_not_matter(cuda, d):
    """NaN in other documents, behind the last document, between the sinks and
    the window, and past the window leaves the results unchanged."""
    lens = [300, 100]
    q, k, v, cq, ck = packed_case(lens, lens, 1, 1, d, BF16, seed=3)
    rule = dict(window=(64, 0), sinks=3, causal=True)
    kk, vv = (torch.cat([t, t[:50]]).to(cuda) for t in (k, v))
    args = (1, d, [0, 20, 120])
    ckk = [0, 300, 400]
    want = ops.attention_window(q[:120].to(cuda), kk, vv, *args, cu_seqlens_k=ckk, **rule)
    for t in (kk, vv):
        t[400:] = float("nan")
        t[10:200] = float("nan")      # the 20 queries of document 0 see 216 .. 299 and 0 .. 2
    got = ops.attention_window(q[:120].to(cuda), kk, vv, *args, cu_seqlens_k=ckk, **rule)
    assert torch.equal(got, want) and torch.isfinite(got).all()
    vv[250, 0] = float("nan")         # a value that they see
    got = ops.attention_window(q[:120].to(cuda), kk, vv, *args, cu_seqlens_k=ckk, **rule)
    assert torch.isnan(got[:20, 0]).all() and torch.equal(got[20:], want[20:])


@pytest.mark.gpu
def test_no_rows_and_no_keys_at_odd_strides(cuda):
    """Empty views keep the strides of what they were cut from."""
    d = 64
    buf = torch.randn(8, d + 3, generator=torch.Generator().manual_seed(7)).to(BF16).to(cuda)
    q = buf[:, :d].contiguous()
    none = buf[:0, 1:1 + d]
    got = ops.attention_window(q, none, none, 1, d, [0, 8], cu_seqlens_k=[0, 0])
    assert got.shape == (8, d) and (got == 0).all()
    assert ops.attention_window(none, q, q, 1, d, [0, 0], cu_seqlens_k=[0, 8]).shape == (0, d)
    assert ops.attention_window(none, none, none, 1, d, [0]).shape == (0, d)
    n = torch.zeros(2, dtype=torch.int32, device=cuda)
    qd = q.view(2, 4, 1, d)
    empty = torch.empty(2, 0, 1, d + 3, dtype=BF16, device=cuda)[..., 1:1 + d]
    got = ops.attention_window_decode(qd, empty, empty, n)
    assert got.shape == qd.shape and (got == 0).all()


@pytest.mark.gpu
def test_strided_views_and_outputs(cuda):
    d, rows = 64, 150
    qkv = torch.randn(rows, 4 * d, generator=torch.Generator().manual_seed(4)).to(BF16).to(cuda)
    q, k, v = qkv.split([2 * d, d, d], 1)
    rule = dict(kv_heads=1, window=(20, 20), sinks=2)
    want = ops.attention_window(q.contiguous(), k.contiguous(), v.contiguous(), 2, d, [0, 100, 140],
                                **rule)
    assert (want[140:] == 0).all()
    out = torch.full((rows, 3 * d), 9.0, dtype=BF16, device=cuda)
    got = ops.attention_window(q, k, v, 2, d, [0, 100, 140], out=out[:, d:], **rule)
    assert torch.equal(got[:140], want[:140])
    assert (out[140:] == 9).all() and (out[:, :d] == 9).all()
    odd = qkv[:, 1:1 + 2 * d]         # rows that are not 16-byte aligned are copied
    assert torch.equal(ops.attention_window(odd, k, v, 2, d, [0, rows], **rule),
                       ops.attention_window(odd.contiguous(), k, v, 2, d, [0, rows], **rule))


# ---------------------------------------------------------------- GPU: single tokens
def check_decode(got, q, k, v, lens, rule):
    B, n, H, d = q.shape
    kv = k.shape[2]
    half = torch.finfo(q.dtype).eps / 2
    for b, length in enumerate(lens):
        see = seen_mask(n, length, *rule)
        for h in range(H):
            m = h // (H // kv)
            want, off = attend(q[b, :, h], k[b, :length, m], v[b, :length, m], see, d ** -0.5, half)
            check(got[b, :, h], want, off)
            assert (got[b, :, h][~see.any(-1)] == 0).all()


def decode_case(lens, room, n, H, kv, d, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    q = (torch.randn(len(lens), n, H, d, generator=g) * 1.5).to(dtype)
    k = torch.randn(len(lens), room, kv, d, generator=g).to(dtype)
    v = torch.randn(len(lens), room, kv, d, generator=g).to(dtype)
    return q, k, v, torch.tensor(lens, dtype=torch.int32)


@pytest.mark.gpu
@pytest.mark.parametrize("rule", RULES)
@pytest.mark.parametrize("n,H,kv,d,dtype", [(1, 7, 1, 128, BF16), (1, 4, 4, 64, F16),
                                            (3, 6, 1, 64, BF16), (2, 20, 2, 128, F16)])
def test_decode(cuda, rule, n, H, kv, d, dtype):
    lens = [0, 1, 2, 15, 16, 17, 300, 777, 1000]
    q, k, v, length = decode_case(lens, 1000, n, H, kv, d, dtype)
    got = ops.attention_window_decode(q.to(cuda), k.to(cuda), v.to(cuda), length.to(cuda),
                                      window=rule[:2], sinks=rule[2], causal=rule[3])
    check_decode(got.cpu(), q, k, v, lens, rule)


@pytest.mark.gpu
@pytest.mark.parametrize("B", [1, 40])
def test_decode_splits(cuda, B):
    """One sequence over a whole cluster, many over one CTA each."""
    lens = [(4001 * (i + 1)) % 4097 for i in range(B)]
    q, k, v, length = decode_case(lens, 4096, 1, 8, 4, 64, BF16, seed=5)
    got = ops.attention_window_decode(q.to(cuda), k.to(cuda), v.to(cuda), length.to(cuda))
    check_decode(got.cpu(), q, k, v, lens, (None, None, 0, True))


@pytest.mark.gpu
def test_decode_cache_layouts_and_unused_rows(cuda):
    q, k, v, length = decode_case([40, 100, 7], 128, 1, 4, 2, 64, F16, seed=6)
    q, k, v, length = (t.to(cuda) for t in (q, k, v, length))
    rule = dict(window=(31, 0), sinks=2)
    want = ops.attention_window_decode(q, k, v, length, **rule)
    by_head = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (k, v)]
    assert torch.equal(ops.attention_window_decode(q, *by_head, length, **rule), want)
    for t in (k, v):                      # rows past each length, and outside the window
        t[0, 40:], t[1, 100:], t[2, 7:] = (float("nan"),) * 3
        t[1, 2:68] = float("nan")
    assert torch.equal(ops.attention_window_decode(q, k, v, length, **rule), want)
    # lengths out of range are clamped to the cache
    far = torch.tensor([1 << 30, -5, 7], dtype=torch.int32, device=cuda)
    k2, v2 = torch.nan_to_num(k), torch.nan_to_num(v)
    full = torch.tensor([128, 0, 7], dtype=torch.int32, device=cuda)
    assert torch.equal(ops.attention_window_decode(q, k2, v2, far, **rule),
                       ops.attention_window_decode(q, k2, v2, full, **rule))


@pytest.mark.gpu
def test_decode_graph_follows_device_lengths(cuda):
    q, k, v, length = decode_case([5, 90], 96, 1, 2, 1, 128, BF16, seed=7)
    q, k, v, length = (t.to(cuda) for t in (q, k, v, length))
    out = torch.empty_like(q)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.attention_window_decode(q, k, v, length, window=(20, 0), sinks=1, out=out)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.attention_window_decode(q, k, v, length, window=(20, 0), sinks=1, out=out)
    for lens in ([5, 90], [96, 0], [33, 41]):
        length.copy_(torch.tensor(lens, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        check_decode(out.cpu(), q.cpu(), k.cpu(), v.cpu(), lens, (20, 0, 1, True))


@pytest.mark.gpu
def test_offsets_beyond_32_bits(cuda):
    """The last keys of 2^31 and more elements, in a cache and in packed rows."""
    room, kv, d, m = 1 << 21, 4, 128, 300
    g = torch.Generator().manual_seed(10)
    tail = torch.randn(m, kv, d, generator=g).to(BF16)
    cache = torch.zeros(2, room + 8, kv, d, dtype=BF16, device=cuda)
    cache[1, room + 8 - m:] = tail.to(cuda)
    q = torch.randn(2, 1, 2 * kv, d, generator=g).to(BF16)
    lens = torch.tensor([1, room + 8], dtype=torch.int32, device=cuda)
    got = ops.attention_window_decode(q.to(cuda), cache, cache, lens, window=(m - 1, 0)).cpu()
    check_decode(got[1:], q[1:], tail[None], tail[None], [m], (m - 1, 0, 0, True))
    rows = cache.view(-1, kv * d)
    end = rows.shape[0]
    qp = torch.randn(70, 2 * kv * d, generator=g).to(BF16)
    got = ops.attention_window(qp.to(cuda), rows, rows, 2 * kv, d, [0, 70], kv_heads=kv,
                               cu_seqlens_k=[end - m, end], window=(100, 0)).cpu()
    t = tail.view(m, kv * d)
    check_packed(got, qp, t, t, [0, 70], [0, m], 2 * kv, kv, d, (100, 0, 0, False))


@pytest.mark.gpu
def test_gpu_refusals(cuda):
    x = torch.zeros(8, 256, dtype=BF16, device=cuda)
    for bad in (dict(heads=2, head_dim=96), dict(heads=3, head_dim=128, kv_heads=2),
                dict(heads=2, head_dim=128, window=(-1, 0)),
                dict(heads=2, head_dim=128, sinks=-1), dict(heads=2, head_dim=128, scale=0.0),
                dict(heads=2, head_dim=128, cu_seqlens=[0, 9]),
                dict(heads=2, head_dim=128, cu_seqlens=[0, 5, 4]),
                dict(heads=2, head_dim=128, cu_seqlens_k=[0, 4, 8]),
                dict(heads=4, head_dim=128)):
        bad = {"cu_seqlens": [0, 8], **bad}
        with pytest.raises(ValueError):
            ops.attention_window(x, x, x, bad.pop("heads"), bad.pop("head_dim"),
                                 bad.pop("cu_seqlens"), **bad)
    with pytest.raises(TypeError):
        ops.attention_window(x, x.half(), x, 2, 128, [0, 8])
    c = torch.zeros(2, 8, 2, 128, dtype=BF16, device=cuda)
    n = torch.zeros(2, dtype=torch.int32, device=cuda)
    q = c[:, :1]
    for args in ((q, c, c, n.long()), (q, c, c, n[:1]), (q[:1], c, c, n), (q, c, c[:, :4], n),
                 (q, c[..., :64], c[..., :64], n), (q, c[:, :, :, ::2], c[:, :, :, ::2], n),
                 (q[0], c, c, n)):
        with pytest.raises(ValueError):
            ops.attention_window_decode(*args)
    with pytest.raises(ValueError):
        ops.attention_window_decode(q, c, c, n, window=(0, -1))
    with pytest.raises(ValueError):      # a cache that would have to be copied
        ops.attention_window_decode(q[..., :64], c.flatten(2)[..., 4:132].unflatten(2, (2, 64)),
                                    c.flatten(2)[..., 4:132].unflatten(2, (2, 64)), n)
    with pytest.raises(TypeError):
        ops.attention_window_decode(q.half(), c, c, n)
