"""Calls of the 4-bit key/value cache that its documentation allows and that lie at the edge of what its kernels divide up."""
import ctypes as C

import numpy as np
import pytest
import torch

import ring_attention_b200 as ra
from ring_attention_b200 import _lib
from tests import cache4_oracle as O
from tests.test_gpu_cache4 import BF16, F32, ROOM, Filled, _i32, _np, _rand

pytestmark = pytest.mark.gpu


def _filled(d, n, k, v, room=ROOM, dtype=BF16, positions=None):
    """A cache of one sequence and head with the rows k, v [n, d] (NumPy), and the values that it stands for."""
    cache = ra.KVCache4(1, 1, room or n, d)
    k, v = (torch.from_numpy(np.asarray(x, np.float32)).cuda().to(dtype).view(1, n, 1, d) for x in (k, v))
    cache.append(k, v, positions=None if positions is None else _i32(positions)[None])
    return cache, O.values(_np(k)[0]), O.values(_np(v)[0])


def _check_rows(q, k, v, kpos, qpos, out, lse, weights, scale, causal=False, form="many"):
    """bf16 calls of one key/value head, with bounds that go by what each query sees and gives weight to.

    A score is formed in fp32 from at most 3 * 16 partial products of a group's codes and its middle; with M the largest |k| of a
    key's group it is off by at most e = 64 * 2^-24 scale sum |q| M + 4 * 2^-24 |s|.  The log-sum-exp is off by sum p e and 2^-21
    and 2^-22 of itself; a probability by the factor 1 + e + that, the result by that of p |v|, by half a step of bf16 and, where
    values are rounded to fp16, by 2^-11 of each and 2^-11 of each p; elsewhere by 2^-11 of p step code <= p (|v| + |min|)."""
    lq, h, d = q.shape
    n = len(k)
    want = O.attend(q, k, v, np.asarray(kpos)[None], qpos, scale, causal=causal)
    vis = np.asarray(kpos)[None] <= np.asarray(qpos)[:, None] if causal else np.ones((lq, n), bool)
    group = np.abs(k[:, 0]).reshape(n, d // 64, 64).max(-1).repeat(64, 1)
    least = np.abs(v[:, 0].reshape(n, d // 64, 64).min(-1)).repeat(64, 1)
    size_v = np.abs(v[:, 0]) + (0 if form == "many" else least)
    total, slack = np.zeros(n), np.zeros(n)
    for i in range(h):
        s = q[:, i] @ k[:, 0].T * scale
        e = 64 * 2.0**-24 * (np.abs(q[:, i]) @ group.T) * scale + 4 * 2.0**-24 * np.abs(s)
        p = np.where(vis, np.exp(np.where(vis, s, -np.inf) - want["lse"][i][:, None]), 0)
        le = (p * e).sum(-1) + 2.0**-21 + 2.0**-22 * np.abs(want["lse"][i])
        err = np.abs(_np(lse)[0, i] - want["lse"][i])
        assert (err <= le).all(), (i, (err / le).max())
        pe = p * (e + le[:, None])
        tol = 2.0**-8 * np.abs(want["out"][:, i]) + 2 * pe @ np.abs(v[:, 0]) + (2.0**-10 * p) @ size_v
        tol += 2.0**-24 * p.max() * np.abs(v[vis.any(0), 0]).max()
        err = np.abs(_np(out)[0, :, i] - want["out"][:, i])
        assert (err <= tol).all(), (i, (err / tol).max())
        total += p.sum(0)
        slack += 2 * pe.sum(0) + 2.0**-20 * p.sum(0)
    w = _np(weights)[0, 0, :n]
    assert (np.abs(w - total) <= slack + lq * h * 2.0**-125 + 2.0**-23 * total).all()


# ---- many query rows: powers of two of the operands -------------------------------------------------------------
@pytest.mark.parametrize("hidden", [True, False])
@pytest.mark.parametrize("zero,loud", [((0, 1), 5), ((5, 6), 0), ((70, 71), 100), ((100, 101), 70), ((3, 4), 130), ((0, 64), 130), ((0, 100), 150),
                                       ((64, 128), 5), ((1, 192), 0)])
@pytest.mark.parametrize("size", [20, 64, 80, 100])
@pytest.mark.parametrize("lq,room", [(70, ROOM), (2, None), (2, ROOM)])
def test_rows_of_zeros_beside_rows_of_any_size(lq, room, size, zero, loud, hidden):
    """Value rows of zeros and one of 2^size in a unit, or units apart; the large one in sight or behind a mask."""
    rng = np.random.default_rng(size + zero[0])
    d, n = 128, 192
    k, v = rng.standard_normal((n, d)), rng.standard_normal((n, d)) + 0.3
    v[zero[0]:zero[1]] = 0
    v[loud] = np.ldexp(rng.standard_normal(d), size)
    pos = np.arange(n)
    pos[loud] = 5000 if hidden else pos[loud]
    cache, kk, vv = _filled(d, n, k, v, room=room, positions=pos)
    q = _rand(rng, (1, lq, 2, d), BF16)
    q_pos = np.full(lq, n)
    form = "many" if lq > 2 else "few"
    for mod in (ra.ScoreMod(causal=True), None):
        if mod is None and hidden:
            continue
        w = torch.zeros_like(cache.weights)
        out, lse = ra.cache_attention(q, cache, q_positions=_i32(q_pos)[None], bias_fn=mod, return_lse=True, weights_out=w)
        _check_rows(_np(q)[0], kk, vv, pos, q_pos, out, lse, w, d**-0.5, causal=mod is not None, form=form)


@pytest.mark.parametrize("hidden", [True, False])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("row,channel,group", [(1, 1, 1), (256, 1, 1), (64, 20, 1), (64, 50, 1), (1, 300, 1), (900, 1, 2.0**-4), (1, 1, 2.0**-12), (1, 1, 2.0**-24),
                                               (900, 1000, 2.0**-9)])
def test_rows_groups_and_channels_that_stand_out(d, row, channel, group, hidden):
    """One row, one channel of all rows or all groups but the first of another size, in sight or behind a mask: the other keys' scores
    and values are as near as ever.  Few keys have the weight, so that roundings do not cancel."""
    rng = np.random.default_rng(int(row + channel))
    n, lq = 320, 70
    k, v = rng.standard_normal((n, d)) + 0.3, rng.standard_normal((n, d)) + 0.3
    for x in (k, v):
        x[:, 64:] *= group
        x[:, 7] *= channel
        x[70] *= row
    pos = np.arange(n)
    pos[70] = 5000 if hidden else 70
    cache, kk, vv = _filled(d, n, k, v, positions=pos)
    for scale in (d**-0.5, 1.0 / channel):
        q = _rand(rng, (1, lq, 1, d), BF16)
        q_pos = np.full(lq, n)
        w = torch.zeros_like(cache.weights)
        out, lse = ra.cache_attention(q, cache, q_positions=_i32(q_pos)[None], bias_fn=ra.ScoreMod(causal=True), return_lse=True, weights_out=w,
                                      sm_scale=scale)
        _check_rows(_np(q)[0], kk, vv, pos, q_pos, out, lse, w, scale, causal=True)


# ---- arrays of the caller's ------------------------------------------------------------------------------------
@pytest.mark.parametrize("d,lq", [(64, 70), (128, 70), (256, 70), (128, 2)])
@pytest.mark.parametrize("off_k,off_v", [(16, 0), (0, 16), (48, 16)])
def test_arrays_on_16_byte_boundaries(d, lq, off_k, off_v):
    """Codes carved out of a pool: every call takes k and v that do not lie on 32-byte boundaries."""
    f = Filled(d, [150, 64], 2, d, BF16, capacity=ROOM)
    q = _rand(f.rng, (2, lq, 4, d), BF16)
    mod = ra.ScoreMod(causal=True, window=90)
    want = [ra.cache_attention(q, f.cache, bias_fn=m, return_lse=True) for m in (None, mod)]
    there = [f.cache.read(150)]
    nbytes = f.cache.k_codes.numel()
    pool = torch.zeros(2 * nbytes + 256, dtype=torch.uint8, device="cuda")
    assert pool.data_ptr() % 32 == 0 and nbytes % 32 == 0
    k, v = pool[off_k:off_k + nbytes], pool[128 + nbytes + off_v:128 + 2 * nbytes + off_v]
    k.copy_(f.cache.k_codes.flatten())
    v.copy_(f.cache.v_codes.flatten())
    f.cache._struct.k, f.cache._struct.v = k.data_ptr(), v.data_ptr()
    got = [ra.cache_attention(q, f.cache, bias_fn=m, return_lse=True) for m in (None, mod)]
    for x, y in zip(want + there, got + [f.cache.read(150)]):
        for i in (0, 1):  # (the same rows see nothing)
            assert torch.equal(torch.isnan(x[i]), torch.isnan(y[i])) and torch.equal(torch.nan_to_num(x[i]), torch.nan_to_num(y[i]))
    f.cache.append(f.k[:, :1], f.v[:, :1])
    f.cache.evict(100)
    assert torch.isfinite(ra.cache_attention(q, f.cache)).all() and ra.device_status() == 0


# ---- rows taken back -------------------------------------------------------------------------------------------
@pytest.mark.parametrize("t", [1, 5, 40])
@pytest.mark.parametrize("evicted", [False, True])
def test_positions_after_drafts_that_branch(t, evicted):
    """Drafts of one tree repeat positions; what is appended in their place goes on behind the rows that stay."""
    rng = np.random.default_rng(t)
    b, hkv, d, n = 4, 2, 64, 30
    cache = ra.KVCache4(b, hkv, 200, d)
    rows = lambda x: [_rand(rng, (b, x, hkv, d), BF16) for _ in range(2)]  # noqa: E731
    cache.append(*rows(n))
    at = n
    if evicted:  # slots are no positions from here on, and the last rows may be gone
        cache.weights.copy_(torch.rand_like(cache.weights))
        cache.evict(20)
        at = 20
    assert cache.seen.tolist() == [n] * b
    # at `n` one branch and its sibling, then the branch's child: positions n, n + 1, n + 1, n + 2
    cache.append(*rows(4), positions=_i32([[n, n + 1, n + 1, n + 2]] * b))
    assert cache.seen.tolist() == [n + 3] * b and cache.lengths.tolist() == [at + 4] * b
    keep = [0, 1, 2, 4]  # drafts that stay: none, the first, the branch, all
    then = [n, n + 1, n + 2, n + 3]
    cache.append(*rows(t), start=_i32([at + x for x in keep]))
    assert cache.lengths.tolist() == [at + x + t for x in keep]
    assert cache.seen.tolist() == [x + t for x in then]
    for i in range(b):
        for j in range(hkv):
            assert cache.positions[i, j, at + keep[i]:at + keep[i] + t].tolist() == list(range(then[i], then[i] + t))
    # no rows in their place: the sequence stands where it stood before the last ones
    cache.append(*rows(t), start=_i32([at + x for x in keep]), counts=_i32([0] * b))
    assert cache.lengths.tolist() == [at + x for x in keep] and cache.seen.tolist() == then
    q = _rand(rng, (b, 1, hkv, d), BF16)
    one = ra.cache_attention(q, cache, bias_fn=ra.ScoreMod(causal=True, window=7))
    want = ra.cache_attention(q, cache, q_positions=_i32([[x - 1] for x in then]), bias_fn=ra.ScoreMod(causal=True, window=7))
    assert torch.equal(torch.nan_to_num(one), torch.nan_to_num(want)) and ra.device_status() == 0


def test_start_in_a_graph_with_more_rows_than_a_block_takes():
    """Replays of a captured append that drops rows: the counters and positions that a replay finds are those of the one before."""
    rng = np.random.default_rng(3)
    cache = ra.KVCache4(2, 1, 200, 64)
    k, v = (_rand(rng, (2, 40, 1, 64), BF16) for _ in range(2))
    start = _i32([10, 0])
    cache.append(k, v)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        cache.append(k, v, start=start)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.append(k, v, start=start)
    for at in ([3, 40], [0, 45], [40, 99]):
        start.copy_(_i32(at))
        before = cache.lengths.tolist()
        graph.replay()
        at = [min(x, n) for x, n in zip(at, before)]
        assert cache.lengths.tolist() == [x + 40 for x in at] == cache.seen.tolist()
        for i in range(2):
            assert cache.positions[i, 0, :at[i] + 40].tolist() == list(range(at[i] + 40))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_no_rows_at_start_drop_what_is_behind(dtype):
    rng = np.random.default_rng(5)
    cache = ra.KVCache4(3, 2, 100, 128)
    k, v = _rand(rng, (3, 30, 2, 128), dtype), _rand(rng, (3, 30, 2, 128), dtype)
    cache.append(k, v)
    was = cache.read(30)
    cache.append(k[:, :0], v[:, :0])  # nothing to add, nothing to drop
    assert cache.lengths.tolist() == [30] * 3
    cache.append(k[:, :0], v[:, :0], start=_i32([7, 0, 99]))
    assert cache.lengths.tolist() == [7, 0, 30] == cache.seen.tolist()
    for x, y in zip(was, cache.read(30)):
        assert torch.equal(x[0, :7], y[0, :7]) and torch.equal(x[2], y[2]) and y[0, 7:].abs().max() == 0
    cache.append(k[:, :1], v[:, :1])
    assert cache.positions[:, 1, :].gather(1, cache.lengths[:, None].long() - 1).flatten().tolist() == [7, 0, 30]


# ---- parts held apart ------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,lq", [(F32, 1), (BF16, 1), (BF16, 70)])
def test_parts_of_a_cache_held_apart_are_joined_by_their_log_sum_exps(dtype, lq):
    """Four parts, as the ranks of a ring hold them; one is empty for the first sequence, others lie outside the window."""
    rng = np.random.default_rng(51)
    b, hkv, h, d, n, parts = 2, 2, 4, 128, 400, 4
    k, v = _rand(rng, (b, n, hkv, d), dtype), _rand(rng, (b, n, hkv, d), dtype)
    q = _rand(rng, (b, lq, h, d), dtype)
    lengths, each = [290, 400], n // parts
    q_pos = np.array([[x - lq + i for i in range(lq)] for x in lengths])
    mod, window = ra.ScoreMod(causal=True, window=130), 130
    outs, lses = [], []
    for i in range(parts):
        cache = ra.KVCache4(b, hkv, 64000, d)
        at = slice(i * each, (i + 1) * each)
        cache.append(k[:, at], v[:, at], counts=_i32([min(max(x - i * each, 0), each) for x in lengths]),
                     positions=torch.arange(i * each, (i + 1) * each, device="cuda").expand(b, each).contiguous())
        out, lse = ra.cache_attention(q, cache, q_positions=_i32(q_pos), bias_fn=mod, return_lse=True)
        outs.append(out.double())
        lses.append(lse.double())
    assert torch.isneginf(lses[3][0]).all() and torch.isneginf(lses[0][0, :, -1]).all() and torch.isnan(outs[3][0]).all()
    L = torch.logsumexp(torch.stack(lses), 0)
    got = torch.zeros_like(outs[0])
    for out, lse in zip(outs, lses):
        share = torch.exp(lse - L).transpose(1, 2)[..., None]
        got += torch.where(share > 0, share * out, torch.zeros_like(out))
    # each part is off by what a call is: (2 es + 2^-20) 2 max |v|, and in bf16 by half a step of its own result and by the
    # roundings of p and of values or p step code, together 2^-8, 2^-10 and 2^-11 * 15 / 8 of the largest value at most
    kk, vv = O.values(_np(k)), O.values(_np(v))
    for i, x in enumerate(lengths):
        want = O.attend(_np(q)[i], kk[i, :x], vv[i, :x], np.tile(np.arange(x), (hkv, 1)), q_pos[i], d**-0.5, causal=True, window=window)
        es = 64 * 2.0**-24 * want["size"] + 4 * 2.0**-24 * want["top"]
        vmax = np.abs(vv[i, :x]).max()
        tol = (2 * es + 2.0**-20)[None, :, None] * 4 * vmax + (0 if dtype == F32 else (2.0**-8 + 2.0**-10 + 2.0**-10) * vmax)
        assert (np.abs(_np(got)[i] - want["out"]) <= tol).all()
        assert (np.abs(_np(L)[i] - want["lse"]) <= 2 * es[:, None] + 2.0**-20 + 2.0**-21 * np.abs(want["lse"])).all()


# ---- weights ---------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("lq,room", [(0, None), (1, None), (70, ROOM)])
def test_weights_of_slots_behind_the_last_row_are_left(lq, room):
    f = Filled(41, [0, 5, 64, 100], 2, 64, BF16, capacity=room)
    f.cache.weights.copy_(torch.rand_like(f.cache.weights))
    w = torch.full_like(f.cache.weights, -3.0)
    q = _rand(f.rng, (4, lq, 2, 64), BF16)
    out = ra.cache_attention(q, f.cache, weights_out=w)
    assert out.shape == q.shape
    for i, n in enumerate(f.lengths):
        assert (w[i, :, n:] == -3.0).all()
        more = w[i, :, :n] - f.cache.weights[i, :, :n]
        assert (more > 0).all() if lq else (more == 0).all()


# ---- NaN under masks -------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,lq,room", [(F32, 2, None), (F32, 2, ROOM), (BF16, 2, None), (BF16, 2, ROOM), (BF16, 40, None), (BF16, 70, ROOM)])
@pytest.mark.parametrize("at", [0, 130, 199])
def test_nan_reaches_rows_that_see_it_however_little_they_weigh_it(dtype, lq, room, at):
    """ALiBi takes the probability of a key far behind the query below what a float holds; its NaN value counts all the same, and
    a key outside the window or behind the query does not."""
    f = Filled(31, [200], 2, 128, dtype, capacity=room)
    v = f.v.clone()
    v[0, at, 1, 70] = float("nan")
    f.cache.append(f.k, v, start=_i32([0]))
    q = _rand(f.rng, (1, lq, 4, 128), dtype)
    slopes = torch.tensor([0.0, 40.0, 0.0, 40.0], device="cuda")
    for window in (0, 150):
        pos = torch.arange(100, 100 + 3 * lq, 3, device="cuda")[None]
        mod = ra.ScoreMod(causal=True, alibi_slopes=slopes, window=window)
        out, lse = ra.cache_attention(q, f.cache, q_positions=pos, bias_fn=mod, return_lse=True)
        sees = (pos[0] >= at) & ((pos[0] - at < window) if window else True)
        for h in range(4):
            bad = torch.zeros(lq, 128, dtype=torch.bool, device="cuda")
            if h >= 2:
                bad[:, 64:] = sees[:, None]
            assert torch.equal(torch.isnan(out[0, :, h]), bad), (window, h)
        assert torch.isfinite(lse).all()


# ---- refusals --------------------------------------------------------------------------------------------------
def test_append_refuses_what_asks_for_a_gradient():
    cache = ra.KVCache4(1, 1, 64, 64)
    x = torch.ones(1, 2, 1, 64, device="cuda")
    y = x.clone().requires_grad_(True)
    for k, v in ((y, x), (x, y), (y * 2, x)):
        with pytest.raises(ra.RingAttentionError):
            cache.append(k, v)
    assert cache.lengths.tolist() == [0]
    with torch.no_grad():
        cache.append(y, y)
    cache.append(y.detach(), x)
    assert cache.lengths.tolist() == [4]


def test_the_status_call_says_what_happened_to_a_full_cache():
    """Bit 17 alone is about dropped rows, not about a wait."""
    cache = ra.KVCache4(1, 1, 64, 64)
    x = torch.ones(1, 40, 1, 64, device="cuda")
    cache.append(x, x)
    cache.append(x, x)
    bits = C.c_uint32(0)
    assert _lib.lib.ra_device_status(C.byref(bits)) == _lib.RA_ERR_DEVICE_STATUS and bits.value == 1 << 17
    text = _lib.lib.ra_last_error_string().decode()
    assert "capacity" in text and "wait" not in text
    assert ra.device_status() == 0
