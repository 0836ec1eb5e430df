"""Operators of a batch of continuations of one prompt (prefix_attention.hip, cache_cut.hip, sampling.hip): attention over shared cells, what cells are given, cuts of a cache, sampling.  Against their definitions in 64 bits."""
import ctypes as C

import numpy as np
import pytest

from pipeinfer_amd import lib as L

P = 4096                                                                       # an address that no refused call looks at


def attention_call(lib, q=P, stride=None, k=P, v=P, mask=P, scale=0.1, dim=64, heads=8, kv=2, tok=3, prompt=100, n=140, scratch=P, floats=1 << 40, out=P, out_stride=None, lse=None, dyn=None, stream=None):
    return lib.pi_op_prefix_attention(q, heads * dim if stride is None else stride, k, v, mask, scale, dim, heads, kv, tok, prompt, n, scratch, floats, out, heads * dim if out_stride is None else out_stride, lse, dyn, stream)


@pytest.mark.parametrize("args,why", [
    (dict(dim=60), b"8 .. 256 values in steps of 8"), (dict(dim=264), b"8 .. 256"), (dict(dim=0), b"8 .. 256"), (dict(kv=3), b"whole groups"), (dict(heads=0), b"0 query heads"), (dict(kv=0), b"over 0 key"),
    (dict(tok=-1), b"-1 tokens"), (dict(prompt=141), b"141 of 140 cells"), (dict(prompt=-1), b"-1 of 140"), (dict(scale=0.0), b"scale 0"), (dict(scale=-1.0), b"scale -1"), (dict(scale=float("nan")), b"scale"),
    (dict(scale=float("inf")), b"scale"), (dict(q=None), b"are NULL"), (dict(k=None), b"are NULL"), (dict(v=None), b"are NULL"), (dict(out=None), b"are NULL"), (dict(mask=None), b"are NULL"), (dict(stride=504), b"504"),
    (dict(stride=516), b"516"), (dict(out_stride=508), b"508"), (dict(out_stride=514), b"514"), (dict(q=P + 8), b"16 bytes"), (dict(k=P + 2), b"16 bytes"), (dict(v=P + 4), b"16 bytes"), (dict(out=P + 4), b"16 bytes"),
    (dict(scratch=None), b"0 floats of scratch"), (dict(floats=10), b"10 floats of scratch"), (dict(scratch=P + 8), b"on 16 bytes, for"),
])
def test_attention_refuses(args, why):
    lib = L.load()
    assert attention_call(lib, **args) != 0 and why in lib.pi_last_error(), lib.pi_last_error()


@pytest.mark.parametrize("call,why", [
    (lambda lib, mass: mass(dim=12), b"steps of 8"), (lambda lib, mass: mass(prompt=500), b"500 of"), (lambda lib, mass: mass(lse=None), b"are NULL"), (lambda lib, mass: mass(mass=None), b"are NULL"),
    (lambda lib, mass: mass(k=None), b"are NULL"), (lambda lib, mass: mass(mask=None), b"are NULL"), (lambda lib, mass: mass(q=P + 2), b"16 bytes"), (lambda lib, mass: mass(stride=511), b"511"), (lambda lib, mass: mass(decay=float("nan")), b"decay"),
    (lambda lib, mass: mass(scale=float("inf")), b"scale"), (lambda lib, mass: mass(scale=0.0), b"scale 0"), (lambda lib, mass: mass(scale=-0.1), b"scale -0.1"), (lambda lib, mass: mass(scratch=None), b"0 floats"), (lambda lib, mass: mass(floats=3), b"3 floats"),
    (lambda lib, mass: lib.pi_op_cache_choose(P, None, 10, 11, P, None), b"11 of 10"), (lambda lib, mass: lib.pi_op_cache_choose(P, None, 10, -1, P, None), b"-1 of 10"), (lambda lib, mass: lib.pi_op_cache_choose(None, None, 10, 4, P, None), b"is NULL"),
    (lambda lib, mass: lib.pi_op_cache_choose(P, None, 10, 4, None, None), b"is NULL"),
    (lambda lib, mass: lib.pi_op_cache_move((C.c_void_p * 1)(P), (C.c_int64 * 1)(16), 1, P, 11, 10, None), b"11 of 10"), (lambda lib, mass: lib.pi_op_cache_move(None, None, 1, P, 4, 10, None), b"is NULL"),
    (lambda lib, mass: lib.pi_op_cache_move((C.c_void_p * 1)(P), (C.c_int64 * 1)(16), 1, P, 0x7fffff00, 0x7fffffff, None), b"2147483392 of"),
    (lambda lib, mass: lib.pi_op_cache_move((C.c_void_p * 1)(0), (C.c_int64 * 1)(16), 1, P, 4, 10, None), b"array 0 is NULL"), (lambda lib, mass: lib.pi_op_cache_move((C.c_void_p * 1)(P), (C.c_int64 * 1)(0), 1, P, 4, 10, None), b"rows of 0 bytes"),
    (lambda lib, mass: lib.pi_op_cache_move((C.c_void_p * 1)(P), (C.c_int64 * 1)(16), 1, None, 4, 10, None), b"is NULL"), (lambda lib, mass: lib.pi_op_cache_move((C.c_void_p * 1)(P), (C.c_int64 * 1)(16), -1, P, 4, 10, None), b"-1 arrays"),
    (lambda lib, mass: lib.pi_op_sample(P, 99, 100, 1, P, P, P, P, P, P, 1 << 30, P, P, P, None), b"99 apart"), (lambda lib, mass: lib.pi_op_sample(P, 100, 0, 1, P, P, P, P, P, P, 1 << 30, P, P, P, None), b"1 .. 524288"),
    (lambda lib, mass: lib.pi_op_sample(P, 1 << 20, 1 << 20, 1, P, P, P, P, P, P, 1 << 30, P, P, P, None), b"1 .. 524288"), (lambda lib, mass: lib.pi_op_sample(P, 100, 100, -1, P, P, P, P, P, P, 1 << 30, P, P, P, None), b"-1 rows"),
    (lambda lib, mass: lib.pi_op_sample(None, 100, 100, 1, P, P, P, P, P, P, 1 << 30, P, P, P, None), b"are NULL"), (lambda lib, mass: lib.pi_op_sample(P, 100, 100, 1, P, P, P, P, None, P, 1 << 30, P, P, P, None), b"are NULL"),
    (lambda lib, mass: lib.pi_op_sample(P, 100, 100, 1, P, P, P, P, P, P, 1 << 30, None, P, P, None), b"are NULL"),
])
def test_the_others_refuse(call, why):
    lib = L.load()

    def mass(q=P, stride=512, k=P, mask=P, lse=P, scale=0.1, dim=64, heads=8, kv=2, tok=3, prompt=100, n=140, decay=1.0, scratch=P, floats=1 << 40, mass=P, dyn=None):
        return lib.pi_op_attention_mass(q, stride, k, mask, lse, scale, dim, heads, kv, tok, prompt, n, decay, scratch, floats, mass, dyn, None)

    assert call(lib, mass) != 0 and why in lib.pi_last_error(), lib.pi_last_error()


def test_nothing_to_do_is_no_error():
    """no tokens, no rows, no arrays, nothing kept or nothing given up: done without a launch (none would succeed here)"""
    lib = L.load()
    assert attention_call(lib, tok=0) == 0 and lib.pi_op_sample(P, 100, 100, 0, P, P, P, P, P, P, 0, P, P, P, None) == 0 and lib.pi_op_cache_choose(P, None, 10, 0, P, None) == 0
    one, size = (C.c_void_p * 1)(P), (C.c_int64 * 1)(16)
    assert lib.pi_op_cache_move(one, size, 0, P, 4, 10, None) == 0 and lib.pi_op_cache_move(one, size, 1, P, 0, 10, None) == 0 and lib.pi_op_cache_move(one, size, 1, P, 10, 10, None) == 0
    assert lib.pi_op_attention_mass(P, 512, P, P, P, 0.1, 64, 8, 2, 0, 100, 140, 1.0, P, 1 << 40, P, None, None) == 0


# ---- on the GPU --------------------------------------------------------------------------------------------------------------------------------------------------------------------
def gpu():
    from tests import gpu_util as U
    return U, U.init()


def pack(seen):
    """[rows][cells] truth values as a bitmap, 32 cells to a word"""
    t, n = seen.shape
    bits = np.zeros((t, (n + 31) // 32 * 32), np.uint8)
    bits[:, :n] = seen
    return np.ascontiguousarray(np.packbits(bits, axis=1, bitorder="little")).view(np.uint32)


def soft_max(q, k, v, seen, scale):
    """out, lse and the weights, [tokens][heads][..], from the definition"""
    T, H, D = q.shape
    per = H // k.shape[1]
    q, k, v = (x.astype(np.float64) for x in (q, k, v))
    out, lse, p = np.zeros((T, H, D)), np.full((T, H), -np.inf), np.zeros((T, H, k.shape[0]))
    for t in range(T):
        c = np.flatnonzero(seen[t])
        if len(c) == 0:
            continue
        for h in range(H):
            s = k[c, h // per] @ q[t, h] * scale
            m = s.max()
            lse[t, h] = m + np.log(np.exp(s - m).sum())
            p[t, h, c] = np.exp(s - lse[t, h])
            out[t, h] = p[t, h, c] @ v[c, h // per]
    return out, lse, p


def inputs(rng, heads, kv, dim, tokens, prompt, own, spread=2.0, loners=True):
    """caches with rows behind the last cell that no call may look at, what nobody sees being no number; token t sees its own cells, the last token no cell behind the prompt"""
    n = prompt + own
    q = (spread * rng.standard_normal((tokens, heads, dim))).astype(np.float16)
    k, v = (rng.standard_normal((n + 5, kv, dim)).astype(np.float16) for _ in range(2))
    seen = np.zeros((tokens, n), bool)
    seen[:, :prompt] = True
    seen[:, prompt:] = rng.random((tokens, own)) < min(1.0, 1.5 / tokens + 0.05)
    if loners:
        seen[-1, prompt:] = False
    nobody = np.append(~seen.any(0), [True] * 5)
    k[nobody], v[nobody] = np.nan, np.inf
    return q, k, v, seen


class Pass:
    """one pass's arrays on the device and its calls; rows of queries and outputs lie further apart than they are long"""

    def __init__(self, U, lib, q, k, v, seen, prompt, scale, room=None):
        self.lib, self.U = lib, U
        self.T, self.H, self.D = q.shape
        self.KH, self.prompt, self.n, self.scale = k.shape[1], prompt, seen.shape[1], scale
        self.qs, self.os = self.H * self.D + 8, self.H * self.D + 4
        rows = np.full((self.T, self.qs), np.nan, np.float16)
        rows[:, :self.H * self.D] = q.reshape(self.T, -1)
        self.room = (prompt, self.n) if room is None else room          # what the arguments say where the device says less
        mask = np.zeros((self.T, max(self.room[1], self.n)), bool)
        mask[:, :self.n] = seen
        mask[:, :prompt] = False                                         # (not looked at)
        self.q, self.k, self.v, self.mask = U.Dev(rows), U.Dev(k), U.Dev(v), U.Dev(pack(mask))
        self.out, self.lse = U.Dev(np.full((self.T, self.os), 7.0, np.float32)), U.Dev(np.full((self.T, self.H), 7.0, np.float32))
        self.dyn = None if room is None else U.Dev(np.array([prompt, self.n], np.int32))
        sizes = (self.D, self.H, self.KH, self.T) + self.room
        self.floats, self.mass_floats = lib.pi_op_prefix_attention_scratch_floats(*sizes), lib.pi_op_attention_mass_scratch_floats(*sizes)
        self.scratch = U.Dev(np.full(max(self.floats, self.mass_floats) + 4, np.nan, np.float32))

    def attend(self, stream=None):
        L.check(self.lib.pi_op_prefix_attention(self.q.ptr, self.qs, self.k.ptr, self.v.ptr, self.mask.ptr, self.scale, self.D, self.H, self.KH, self.T, *self.room, self.scratch.ptr, self.floats, self.out.ptr, self.os, self.lse.ptr,
                                                self.dyn and self.dyn.ptr, stream), "pi_op_prefix_attention")

    def give(self, mass, decay, stream=None):
        L.check(self.lib.pi_op_attention_mass(self.q.ptr, self.qs, self.k.ptr, self.mask.ptr, self.lse.ptr, self.scale, self.D, self.H, self.KH, self.T, *self.room, decay, self.scratch.ptr, self.mass_floats, mass.ptr,
                                              self.dyn and self.dyn.ptr, stream), "pi_op_attention_mass")

    def outputs(self):
        out = self.out.get(np.float32, (self.T, self.os))
        assert (out[:, self.H * self.D:] == 7.0).all()
        assert np.isnan(self.scratch.get(np.float32)[max(self.floats, self.mass_floats):]).all()
        return out[:, :self.H * self.D].reshape(self.T, self.H, self.D), self.lse.get(np.float32, (self.T, self.H))


# A weight's relative error: the score s scale log2(e), |.| < 2^5 here, is rounded at 2^-24 of itself three times (the sum of products, the factor, the difference): 3 x 2^-20 ln 2 = 2e-6 at most, the exponential 2^-23, its two halves 2^-22.
# Sums of n terms in fp32, a few partial sums each of at most 2^11: random signs, 2^-24 x 2^5.5.  An output's error relative to the outputs' size is below the weights' worst one: 4e-6 in the 2-norm
FAR, LSE_FAR = 4e-6, 1e-5


def check_attention(got, want, lse, want_lse):
    assert np.isfinite(got).all()
    assert np.linalg.norm(got - want) <= FAR * np.linalg.norm(want) + 1e-30
    none = np.isneginf(want_lse)
    assert (np.isneginf(lse) == none).all() and (got[none] == 0).all()
    assert np.abs(lse[~none] - want_lse[~none]).max(initial=0.0) <= LSE_FAR                # (at most 2^4: its own rounding is 2^-21, the sum's and the logarithm's as much)


SIZES = [(1, 1, 8, 1, 1, 0), (1, 1, 8, 1, 0, 1), (2, 1, 8, 2, 31, 3), (32, 4, 64, 1, 500, 13), (4, 4, 128, 24, 100, 70), (8, 1, 128, 16, 129, 40), (64, 8, 128, 3, 1000, 33), (71, 1, 64, 2, 65, 90), (71, 1, 64, 1, 0, 700), (6, 2, 40, 33, 64, 1),
         (3, 3, 80, 5, 300, 0), (24, 3, 96, 9, 1, 257), (8, 2, 256, 7, 90, 63), (8, 2, 256, 17, 400, 64), (5, 1, 24, 20, 777, 500), (4, 2, 192, 40, 333, 31), (2, 2, 160, 2, 0, 0), (9, 3, 72, 30, 0, 200), (16, 2, 64, 8, 4096, 64), (4, 1, 32, 64, 2000, 9000)]


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv,dim,tokens,prompt,own", SIZES)
def test_attention(heads, kv, dim, tokens, prompt, own):
    """one token to many, heads with keys of their own to 71 over one, nothing shared, nothing but shared, cells that are no multiple of anything, a token that sees nothing"""
    U, lib = gpu()
    rng = np.random.default_rng(heads * 1000 + tokens)
    q, k, v, seen = inputs(rng, heads, kv, dim, tokens, prompt, own)
    p = Pass(U, lib, q, k, v, seen, prompt, dim ** -0.5)
    p.attend()
    got, lse = p.outputs()
    want, want_lse, _ = soft_max(q, k, v, seen, dim ** -0.5)
    check_attention(got, want, lse, want_lse)


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv,dim,tokens,prompt,own", [(32, 32, 24, 70, 333, 90), (32, 32, 64, 70, 129, 40), (32, 32, 80, 70, 31, 300), (32, 32, 128, 70, 100, 70), (32, 32, 160, 70, 65, 33), (32, 32, 256, 67, 90, 63), (32, 32, 40, 70, 1, 257),
                                                             (32, 32, 64, 70, 0, 50), (32, 32, 96, 129, 97, 0), (16, 16, 128, 128, 300, 20)])
def test_attention_of_many_rows(heads, kv, dim, tokens, prompt, own):
    """as many workgroups as go by 128 rows; the same with sizes that the device knows, and scores far apart"""
    U, lib = gpu()
    rng = np.random.default_rng(dim)
    q, k, v, seen = inputs(rng, heads, kv, dim, tokens, prompt, own)
    want, want_lse, _ = soft_max(q, k, v, seen, dim ** -0.5)
    for room in (None, (prompt + 500, prompt + own + 900)):
        if room:
            k, v = (np.concatenate([x, np.full((room[1] - len(x), kv, dim), np.nan, np.float16)]) for x in (k, v))
        p = Pass(U, lib, q, k, v, seen, prompt, dim ** -0.5, room)
        p.attend()
        got, lse = p.outputs()
        check_attention(got, want, lse, want_lse)
    q[...] = 1.0
    for slope in (0.5, 40.0):
        k[:prompt] = (np.arange(prompt)[:, None, None] * (slope / dim)).astype(np.float16)
        p = Pass(U, lib, q, k, v, seen, prompt, 1.0, room)
        p.attend()
        got, lse = p.outputs()
        want, want_lse, _ = soft_max(q, k, v, seen, 1.0)
        # (scores of up to 2^14: the factor log2(e) and the difference are rounded at 2^-24 of them, the sum of dim <= 256 equal products of 11 bits is exact)
        far = 2 ** -24 * 3 * max(1.0, np.abs(want_lse[np.isfinite(want_lse)]).max())
        assert np.linalg.norm(got - want) <= max(FAR, far) * np.linalg.norm(want) and (np.isneginf(lse) == np.isneginf(want_lse)).all()
        some = np.isfinite(want_lse)
        assert np.abs(lse[some] - want_lse[some]).max(initial=0.0) <= max(LSE_FAR, far)


@pytest.mark.gpu
@pytest.mark.parametrize("prompt,own", [(0, 1 << 20), (1 << 20, 0), (600000, 500000)])
def test_a_million_cells_of_one_head(prompt, own):
    """as many parts of a row as there can be; the values are positive, so that an output's error is the weights'"""
    U, lib = gpu()
    rng = np.random.default_rng(own + 1)
    q, k, _, seen = inputs(rng, 1, 1, 8, 1, prompt, own, loners=False)
    k = np.nan_to_num(k)
    v = (0.5 + rng.random(k.shape)).astype(np.float16)
    seen[:] = True
    p = Pass(U, lib, q, k, v, seen, prompt, 8 ** -0.5)
    p.attend()
    got, lse = p.outputs()
    want, want_lse, _ = soft_max(q, k, v, seen, 8 ** -0.5)
    check_attention(got, want, lse, want_lse)


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv,dim,tokens,prompt,own", [(32, 4, 64, 4, 500, 40), (8, 2, 128, 50, 300, 100)])
def test_sizes_on_the_device(heads, kv, dim, tokens, prompt, own):
    """room for more cells than there are: the device says how many are shared and live; parts without a cell count for nothing, and the mass of what is not live stays"""
    U, lib = gpu()
    rng = np.random.default_rng(tokens)
    for share, live in ((prompt, own), (0, own), (prompt, 0), (prompt // 3, 2 * own), (0, 0)):
        q, k, v, seen = inputs(rng, heads, kv, dim, tokens, share, live)
        room = (4000, 9000)
        k, v = (np.concatenate([x, np.full((room[1] - len(x), kv, dim), np.nan, np.float16)]) for x in (k, v))
        p = Pass(U, lib, q, k, v, seen, share, dim ** -0.5, room)
        p.attend()
        got, lse = p.outputs()
        want, want_lse, w = soft_max(q, k, v, seen, dim ** -0.5)
        check_attention(got, want, lse, want_lse)
        mass = U.Dev(np.full(room[1], 3.0, np.float32))
        p.give(mass, 0.5)
        m = mass.get(np.float32)
        n = share + live
        assert (m[n:] == 3.0).all() and np.allclose(m[:n], 1.5 + w.sum((0, 1))[:n], rtol=1e-5, atol=1e-5)


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv,dim", [(32, 4, 64), (8, 8, 128), (31, 1, 40)])
def test_one_token_behind_a_short_prompt(heads, kv, dim):
    """the shared and the own cells by the same workgroup: nothing shared, all own ones, gaps, a mask that leaves none, sizes that the device knows"""
    U, lib = gpu()
    rng = np.random.default_rng(heads)
    for prompt, own, live, density, room in ((250, 200, 200, 0.5, None), (1, 256, 256, 1.0, None), (256, 1, 1, 1.0, None), (100, 33, 33, 0.0, None), (0, 5, 5, 1.0, (250, 400)), (77, 100, 100, 0.3, (250, 400)), (250, 0, 0, 1.0, (250, 400)),
                                             (0, 300, 300, 0.2, (250, 400)), (0, 0, 0, 1.0, (250, 400))):
        q, k, v, seen = inputs(rng, heads, kv, dim, 1, prompt, own, loners=False)
        k, v = np.nan_to_num(k), np.nan_to_num(v, posinf=1.0)
        seen[:, prompt:] = rng.random((1, own)) < density
        if room:
            k, v = (np.concatenate([x, np.full((room[1] - len(x), kv, dim), np.nan, np.float16)]) for x in (k, v))
        p = Pass(U, lib, q, k, v, seen, prompt, dim ** -0.5, room)
        p.attend()
        got, lse = p.outputs()
        want, want_lse, _ = soft_max(q, k, v, seen, dim ** -0.5)
        check_attention(got, want, lse, want_lse)


@pytest.mark.gpu
def test_nothing_but_the_prompt_by_the_arguments():
    """without a mask, the prompt's end inside a word; the device says that less is shared: the mask counts then, and without one nothing behind the prompt is there"""
    U, lib = gpu()
    rng = np.random.default_rng(23)
    for tokens, room in ((1, 300), (3, 300), (40, 777)):
        for prompt, n in ((room, room), (room - 90, room - 20), (0, 70), (37, 37)):
            q, k, v, seen = inputs(rng, 8, 2, 64, tokens, prompt, n - prompt)
            k, v = np.nan_to_num(k), np.nan_to_num(v, posinf=1.0)
            k, v = (np.concatenate([x, np.zeros((room, 2, 64), np.float16)])[:room] for x in (k, v))
            for masked in (True, False):
                sees = seen.copy()
                if not masked:
                    sees[:, prompt:] = False
                p = Pass(U, lib, q, k, v, sees, prompt, 0.125, (room, room))
                if not masked:
                    p.mask.ptr = None
                p.attend()
                got, lse = p.outputs()
                want, want_lse, w = soft_max(q, k[:n], v[:n], sees, 0.125)
                check_attention(got, want, lse, want_lse)
                mass = U.Dev(np.full(room, 3.0, np.float32))
                p.give(mass, 1.0)
                m = mass.get(np.float32)
                assert (m[n:] == 3.0).all() and np.allclose(m[:n], 3.0 + w.sum((0, 1))[:n], rtol=1e-5, atol=1e-5)


@pytest.mark.gpu
def test_scores_far_apart():
    """scores that grow along the cells by far more than the maximum may lag, that fall, and that are huge: the sums are relative to the right maximum"""
    U, lib = gpu()
    rng = np.random.default_rng(5)
    for tokens in (2, 40):
        for slope in (0.5, -0.5, 40.0):
            q, k, v, seen = inputs(rng, 4, 1, 64, tokens, 700, 50)
            q[...] = 1.0
            k[:750] = (np.arange(750)[:, None, None] * (slope / 64)).astype(np.float16)
            v[:750] = rng.standard_normal((750, 1, 64)).astype(np.float16)
            p = Pass(U, lib, q, k, v, seen, 700, 1.0)
            p.attend()
            got, lse = p.outputs()
            want, want_lse, _ = soft_max(q, k, v, seen, 1.0)
            # (scores of up to 2^15: the sum of products is exact, the factor log2(e) is rounded at 2^-24 of it: 2^-9 x ln 2 of a weight, and of the lse)
            far = 2 ** -24 * 3 * max(1.0, np.abs(want_lse[np.isfinite(want_lse)]).max())
            assert np.linalg.norm(got - want) <= max(FAR, far) * np.linalg.norm(want) and np.abs(lse - want_lse).max() <= max(LSE_FAR, far)


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv,dim,tokens,prompt,own", SIZES)
def test_mass(heads, kv, dim, tokens, prompt, own):
    """what the cells are given adds up to the rows that see anything; the old mass fades, or is not looked at"""
    U, lib = gpu()
    rng = np.random.default_rng(heads * 1000 + tokens + 1)
    q, k, v, seen = inputs(rng, heads, kv, dim, tokens, prompt, own)
    n, scale = prompt + own, dim ** -0.5
    if n == 0:
        return
    p = Pass(U, lib, q, k, v, seen, prompt, scale)
    _, want_lse, w = soft_max(q, k, v, seen, scale)
    p.lse = U.Dev(want_lse.astype(np.float32))
    old = rng.random(n + 3).astype(np.float32)
    given = w.sum((0, 1))[:n]
    for decay, before in ((1.0, old), (0.25, old), (0.0, np.full(n + 3, np.nan, np.float32))):
        mass = U.Dev(before)
        p.give(mass, decay)
        got = mass.get(np.float32)
        want = given + (decay * before[:n].astype(np.float64) if decay else 0.0)
        # (a weight as in FAR, and the lse's own rounding, 2^-21; all terms are positive)
        assert np.allclose(got[:n], want, rtol=8e-6, atol=1e-12), (decay, np.abs(got[:n] / want - 1).max())
        assert np.array_equal(got[n:], before[n:], equal_nan=True)


def chosen(mass, guarded, keep):
    order = sorted(range(len(mass)), key=lambda i: (0, 0, 0, i) if guarded[i] else (1, np.isnan(mass[i]), 0 if np.isnan(mass[i]) else -mass[i], i))[:keep]
    stays = set(order)
    movers = iter(sorted(i for i in order if i >= keep))
    return np.array([i if i in stays else next(movers) for i in range(keep)], np.int32)


@pytest.mark.gpu
@pytest.mark.parametrize("cells", [1, 2, 63, 65, 1000, 4097, 20000, 33000, 100001, 131072, 140001])
def test_choice(cells):
    """masses of every kind: spread, all equal, few different ones, signs, infinities and what is no number; guards, more of them than stay; one cell to all of them"""
    U, lib = gpu()
    rng = np.random.default_rng(cells)
    kinds = {"spread": rng.random(cells) ** 4 * 50, "equal": np.full(cells, 2.5), "few": rng.integers(0, 3, cells) * 0.5, "signs": np.where(rng.random(cells) < 0.3, -0.0, rng.standard_normal(cells)),
             "odd": np.where(rng.random(cells) < 0.2, np.nan, np.where(rng.random(cells) < 0.2, np.inf, np.where(rng.random(cells) < 0.2, -np.inf, rng.standard_normal(cells)))), "zeros": np.where(rng.random(cells) < 0.5, 0.0, -0.0)}
    for name, mass in kinds.items():
        mass = mass.astype(np.float32)
        for keep in sorted({1, cells // 3, cells // 2 + 1, cells - 1, cells} - {0} if cells < 30000 else {cells // 2, 5, cells - 7}):
            if keep == 0:
                continue
            for guards in (None, 0.05, 0.9):
                guarded = np.zeros(cells, bool) if guards is None else rng.random(cells) < guards
                m, g, s = U.Dev(mass), U.Dev(pack(guarded[None])), U.Dev(np.full(keep + 1, -9, np.int32))
                L.check(lib.pi_op_cache_choose(m.ptr, None if guards is None else g.ptr, cells, keep, s.ptr, None), "pi_op_cache_choose")
                got = s.get(np.int32)
                assert np.array_equal(got[:keep], chosen(mass, guarded, keep)) and got[keep] == -9, (name, keep, guards)


@pytest.mark.gpu
@pytest.mark.parametrize("cells,keep,sizes", [(1000, 700, [4, 512, 2064, 6, 1, 16384, 12]), (300, 20, [2048] * 130 + [4]), (5000, 2500, [160, 80, 4]), (400, 250, [65536, 16384, 70000, 2]), (3001, 1500, [8192, 512])])
def test_rows_that_move(cells, keep, sizes):
    """rows of every alignment, more arrays than a launch takes; entries that point in front of the budget or behind the cache move nothing"""
    U, lib = gpu()
    rng = np.random.default_rng(cells)
    source = chosen(rng.random(cells), np.zeros(cells, bool), keep)
    odd = rng.permutation(keep)[:3]
    source[odd] = [0, -5, cells]
    arrays = [rng.integers(0, 256, (cells, b), np.uint8) for b in sizes]
    dev, s = [U.Dev(a) for a in arrays], U.Dev(source)
    at, size = (C.c_void_p * len(dev))(*[d.ptr for d in dev]), (C.c_int64 * len(dev))(*sizes)
    L.check(lib.pi_op_cache_move(at, size, len(dev), s.ptr, keep, cells, None), "pi_op_cache_move")
    for d, a in zip(dev, arrays):
        want = a.copy()
        for i, c in enumerate(source):
            if keep <= c < cells:
                want[i] = a[c]
        assert np.array_equal(d.get(np.uint8, a.shape), want)


def sampled(x, temp, top_k, top_p, min_p, u, clear=1e-9):
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    order = np.argsort(-x, kind="stable")
    order = order[x[order] > -np.inf]
    if len(order) == 0:
        return -1, 0.0, 0, True
    top = x[order[0]]

    def below(v):
        return np.where(v == top, 0.0, v - top)

    if top_k > 0:
        order = order[:top_k]
    w = np.exp(below(x[order]))
    sure = True
    if top_p < 1:
        ahead = np.cumsum(w) - w
        edge = np.float64(top_p) * w.sum()
        n = max(1, int((ahead < edge).sum()))
        near = np.abs(ahead / edge - 1).min() if edge > 0 else 1.0
        sure &= bool(near > clear or top_p <= 0)
        order, w = order[:n], w[:n]
    n = max(1, int((w >= np.float64(min_p)).sum())) if min_p > 0 else len(order)
    order = order[:n]
    if not temp > 0:
        return order[0], 1.0, n, sure
    ids = np.sort(order)
    e = np.exp(below(x[ids]) / np.float64(temp))
    cum = np.cumsum(np.floor(e * 2.0 ** 44 + 0.5))                      # (the steps in which sums are held: weights below half of one are never drawn)
    i = int(np.searchsorted(cum, np.float64(u) * cum[-1], side="right"))
    sure &= bool(np.abs(cum / cum[-1] - u).min() > 1e-9 or u == 0)
    cum = np.cumsum(e)
    return ids[i], e[i] / cum[-1], n, sure


def run_sample(U, lib, x, vocab, settings, u):
    """rows as they are in memory (x: [rows][stride])"""
    rows = len(x)
    size = lib.pi_op_sample_scratch_bytes(vocab, rows)
    d, scratch = U.Dev(x), U.Dev(nbytes=size + 16)
    dev = [None if s is None else U.Dev(np.asarray(s, t)) for s, t in zip(settings, (np.float32, np.int32, np.float32, np.float32))]
    du, out = U.Dev(np.asarray(u, np.float32)), [U.Dev(np.full(rows, -7, t)) for t in (np.int32, np.float32, np.int32)]
    L.check(lib.pi_op_sample(d.ptr, x.shape[1], vocab, rows, *[s and s.ptr for s in dev], du.ptr, scratch.ptr, size, *[o.ptr for o in out], None), "pi_op_sample")
    return [o.get(t) for o, t in zip(out, (np.int32, np.float32, np.int32))]


def check_sample(U, lib, x, vocab, settings, u, clear=1e-9):
    got = run_sample(U, lib, x, vocab, settings, u)
    full = [np.full(len(x), v) if s is None else np.asarray(s) for s, v in zip(settings, (1.0, 0, 1.0, 0.0))]
    for t in range(len(x)):
        i, p, n, sure = sampled(x[t, :vocab], np.float32(full[0][t]), int(full[1][t]), np.float32(full[2][t]), np.float32(full[3][t]), np.float32(u[t]), clear)
        assert sure, ("an input at a border", t)                         # (no test asks which side of a border a sum falls that two roundings could move)
        assert got[0][t] == i and got[2][t] == n and abs(got[1][t] - p) <= 2.0 ** -23 * p, (t, [f[t] for f in full], u[t], got[0][t], i, got[2][t], n, got[1][t], p)


@pytest.mark.gpu
@pytest.mark.parametrize("vocab,stride", [(1, 1), (3, 7), (300, 300), (1000, 1004), (8191, 8191), (32000, 32000), (32001, 32003), (131072, 131072), (262144, 262144), (300001, 300001)])
def test_sample(vocab, stride):
    """every setting by itself and together, the smallest vocabulary to more than most have, rows that begin anywhere"""
    U, lib = gpu()
    rng = np.random.default_rng(vocab)
    rows = 24 if vocab < 100000 else 8
    for spread in (2.5, 8.0):
        x = np.full((rows, stride), np.nan, np.float32)
        x[:, :vocab] = spread * rng.standard_normal((rows, vocab))
        x[::3, :vocab][rng.random(x[::3, :vocab].shape) < 0.6] = -np.inf
        x[:, vocab:] = 100.0
        u = rng.random(rows)
        check_sample(U, lib, x, vocab, (None, None, None, None), u)
        check_sample(U, lib, x, vocab, (np.full(rows, 0.7), np.full(rows, 40), None, None), u)
        check_sample(U, lib, x, vocab, (np.full(rows, 1.3), None, np.full(rows, 0.9), None), u)
        check_sample(U, lib, x, vocab, (None, None, None, np.full(rows, 0.05)), u)
        check_sample(U, lib, x, vocab, (rng.choice([0.0, 0.5, 1.0, 2.0, -1.0], rows), rng.choice([0, 1, 2, 50, 128, 129, 1000, 200000, -3], rows), rng.choice([0.0, 0.3, 0.8, 0.99, 1.0, 2.0], rows), rng.choice([0.0, 0.02, 0.3, 1.0], rows)), u)


@pytest.mark.gpu
@pytest.mark.parametrize("spread", [0.01, 0.1, 0.5, 1.0, 2.0])
def test_sample_of_flat_rows(spread):
    """logits that lie close together, a few far above them, in front or behind, or two crowds; the border among them"""
    U, lib = gpu()
    rng = np.random.default_rng(int(spread * 100))
    V = 100001
    x = (spread * rng.standard_normal((8, V))).astype(np.float32)
    x[1, 90000] += 30 * spread
    x[2, 5] += 20 * spread
    x[3, 50000:50100] += 9 * spread
    x[4, ::2] -= 12 * spread
    x[5, 2000:] -= 30 * spread
    x[6] += 1000.0
    x[7, rng.random(V) < 0.9] = -np.inf
    x[7, :1100] = -np.inf
    # (Weights here are off by 1.4e-13 of themselves, the first term that their series leaves out, and a few 2^-53; a sum by that and by 2^-45 for each of its 200 runs, relative to a total of 1 and more: 6e-12 at most.  numpy's own sums of
    # 100001 terms: 17 halvings x 2^-53 and, one after the other, 10^5 x 2^-53 = 1.1e-11 in cumsum at the very worst, its square root's part as a rule.  The weights at the border of 0.9999 are 1e-8 of the total: 2e-11 keeps clear of both)
    for p in (0.3, 0.95, 0.9999):
        check_sample(U, lib, x, V, (np.full(8, 0.9), None, np.full(8, p), None), rng.random(8), 2e-11)
    check_sample(U, lib, x, V, (None, np.full(8, 700), np.full(8, 0.9), None), rng.random(8))


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [8400, 9000, 16500, 20001, 31000, 32769, 33000, 40960, 40961, 50000, 250000, 524287, 524288])
def test_sample_of_the_few_best(vocab):
    """rows whose last part is short, the best in front, behind and where parts meet, allowed ids in one place, fewer than are asked for"""
    U, lib = gpu()
    rng = np.random.default_rng(vocab)
    x = (2.5 * rng.standard_normal((8, vocab))).astype(np.float32)
    x[1, :vocab - 300] = -np.inf
    x[2, :8000] = x[2, 8400:] = -np.inf
    x[3, vocab - 8300:vocab - 8100] += 20
    x[4] = -np.inf; x[4, rng.integers(0, vocab, 5)] = 1.0
    x[5, -1] = x[5, 0] = x[5, 8191] = x[5, 8192] = x[5].max() + 1
    x[6, rng.random(vocab) < 0.97] = -np.inf
    x[7, vocab // 8192 * 8192 - 60:][:120] += 15
    for k in (1, 2, 20, 100, 128):
        check_sample(U, lib, x, vocab, (np.full(8, 0.8), np.full(8, k), None, None), rng.random(8))
    check_sample(U, lib, x, vocab, (np.full(8, 1.1), np.full(8, 64), np.full(8, 0.9), np.full(8, 0.01)), rng.random(8))


@pytest.mark.gpu
def test_sample_of_odd_rows():
    """rows of equal logits (the border inside them goes by the id), of few values, of nothing, with infinities and what is no number, one logit far above; the ends of u"""
    U, lib = gpu()
    rng = np.random.default_rng(3)
    V = 40000
    x = np.zeros((12, V), np.float32)
    x[1] = rng.integers(-3, 3, V)
    x[2] = -np.inf
    x[3] = np.nan
    x[4] = rng.standard_normal(V); x[4, [7, 900, 39999]] = np.inf
    x[5] = rng.standard_normal(V); x[5, ::2] = np.nan
    x[6] = rng.standard_normal(V); x[6, 123] = 500.0
    x[7] = -np.inf; x[7, 31111] = -3e38
    x[8] = np.where(rng.random(V) < 0.5, 0.0, -0.0)
    x[9] = 1e-30 * rng.standard_normal(V)
    x[10] = 3e38 * np.clip(rng.standard_normal(V), -1, 1)
    x[11] = np.sort(3 * rng.standard_normal(V))
    rows = len(x)
    for u in (0.0, 0.3, 0.777, 1 - 2.0 ** -24):
        for settings in ((None, None, None, None), (np.full(rows, 0.5), np.full(rows, 100), np.full(rows, 0.3), None), (None, np.full(rows, 777), None, None), (None, np.full(rows, 777), np.full(rows, 0.4321), np.full(rows, 0.5)),
                         (None, None, np.full(rows, 0.6543), None), (np.zeros(rows), None, np.full(rows, 0.2), None), (np.full(rows, np.inf), None, None, np.full(rows, 0.01)), (np.full(rows, 1e-3), np.full(rows, 3), None, None)):
            got = run_sample(U, lib, x, V, settings, [u] * rows)
            full = [np.full(rows, v) if s is None else np.asarray(s) for s, v in zip(settings, (1.0, 0, 1.0, 0.0))]
            for t in range(rows):
                with np.errstate(invalid="ignore"):
                    i, p, n, sure = sampled(x[t], np.float32(full[0][t]), int(full[1][t]), np.float32(full[2][t]), np.float32(full[3][t]), np.float32(u))
                if not sure:                                                 # (equal weights put borders on whole counts: u x 40000 may be one.  Then the neighbour is as right)
                    assert abs(int(got[2][t]) - n) <= 1 and abs(got[1][t] - p) <= 1e-4 * p, (t, u)
                    continue
                assert got[0][t] == i and got[2][t] == n and abs(got[1][t] - p) <= 2.0 ** -23 * p, (t, u, got[0][t], i, got[2][t], n, got[1][t], p)


@pytest.mark.gpu
def test_outputs_that_nobody_wants():
    U, lib = gpu()
    rng = np.random.default_rng(8)
    x, ids = U.Dev(rng.standard_normal((3, 500)).astype(np.float32)), [U.Dev(np.zeros(3, np.int32)) for _ in range(2)]
    prob, kept, u = U.Dev(np.zeros(3, np.float32)), U.Dev(np.zeros(3, np.int32)), U.Dev(np.full(3, 0.4, np.float32))
    size = lib.pi_op_sample_scratch_bytes(500, 3)
    scratch = U.Dev(nbytes=size + 16)
    L.check(lib.pi_op_sample(x.ptr, 500, 500, 3, None, None, None, None, u.ptr, scratch.ptr, size, ids[0].ptr, None, None, None), "pi_op_sample")
    L.check(lib.pi_op_sample(x.ptr, 500, 500, 3, None, None, None, None, u.ptr, scratch.ptr, size, ids[1].ptr, prob.ptr, kept.ptr, None), "pi_op_sample")
    assert np.array_equal(ids[0].get(np.int32), ids[1].get(np.int32)) and (kept.get(np.int32) == 500).all()
    q, k, v, seen = inputs(rng, 4, 2, 64, 3, 50, 20)
    p = Pass(U, lib, q, k, v, seen, 50, 0.125)
    p.attend()
    want, _ = p.outputs()
    p.out = U.Dev(np.full((3, p.os), 7.0, np.float32))
    L.check(lib.pi_op_prefix_attention(p.q.ptr, p.qs, p.k.ptr, p.v.ptr, p.mask.ptr, p.scale, 64, 4, 2, 3, 50, 70, p.scratch.ptr, p.floats, p.out.ptr, p.os, None, None, None), "pi_op_prefix_attention")
    assert np.array_equal(p.outputs()[0], want)


@pytest.mark.gpu
def test_a_serving_step():
    """as they are used together: attention, what the cells were given, a cut of the caches, attention over what is left - the same as over the kept cells from the start -, and a token for every row"""
    U, lib = gpu()
    rng = np.random.default_rng(77)
    heads, kv, dim, tokens, prompt, own, scale = 16, 2, 64, 12, 700, 60, 0.125
    n, keep = prompt + own, 400
    q, k, v, seen = inputs(rng, heads, kv, dim, tokens, prompt, own, loners=False)
    k[n:], v[n:] = 0, 0
    bad = ~seen.any(0)
    k[:n][bad], v[:n][bad] = 0, 0
    p = Pass(U, lib, q, k, v, seen, prompt, scale)
    mass = U.Dev(np.zeros(n, np.float32))
    guarded = np.zeros(n, bool)
    guarded[prompt:] = True                                              # the continuations' own cells and the prompt's first
    guarded[:4] = True
    guard, source, pos = U.Dev(pack(guarded[None])), U.Dev(np.zeros(keep, np.int32)), U.Dev(np.arange(n, dtype=np.int32))
    p.attend()
    p.give(mass, 1.0)
    L.check(lib.pi_op_cache_choose(mass.ptr, guard.ptr, n, keep, source.ptr, None), "pi_op_cache_choose")
    arrays = (C.c_void_p * 3)(p.k.ptr, p.v.ptr, pos.ptr)
    L.check(lib.pi_op_cache_move(arrays, (C.c_int64 * 3)(2 * kv * dim, 2 * kv * dim, 4), 3, source.ptr, keep, n, None), "pi_op_cache_move")
    _, _, w = soft_max(q, k, v, seen, scale)
    got_mass, src = mass.get(np.float32), source.get(np.int32)
    assert np.allclose(got_mass, w.sum((0, 1))[:n], rtol=1e-5, atol=1e-9)
    assert np.array_equal(src, chosen(got_mass, guarded, keep)) and np.array_equal(pos.get(np.int32)[:keep], src)
    # the kept cells' mask; how many of them in front everybody still sees
    left = seen[:, src]
    shared = int(np.argmin(left.all(0))) if not left.all() else keep
    after = Pass(U, lib, q, p.k.get(np.float16, k.shape)[:keep + 5], p.v.get(np.float16, v.shape)[:keep + 5], left, shared, scale)
    after.attend()
    out, lse = after.outputs()
    want, want_lse, _ = soft_max(q, k[src], v[src], left, scale)
    check_attention(out, want, lse, want_lse)
    check_sample(U, lib, out.reshape(tokens, -1) * 20, heads * dim, (np.full(tokens, 0.8), np.full(tokens, 40), np.full(tokens, 0.95), np.full(tokens, 0.01)), rng.random(tokens))


class Hip:
    """streams and graphs of the runtime that the library runs on"""

    def __init__(self):
        self.hip = C.CDLL("libamdhip64.so.7")
        for name in ("hipStreamCreate", "hipStreamDestroy", "hipStreamBeginCapture", "hipStreamEndCapture", "hipGraphInstantiate", "hipGraphLaunch", "hipGraphExecDestroy", "hipGraphDestroy"):
            getattr(self.hip, name).restype = C.c_int

    def stream(self):
        s = C.c_void_p()
        assert self.hip.hipStreamCreate(C.byref(s)) == 0
        return s.value

    def capture(self, stream, work):
        graph, run = C.c_void_p(), C.c_void_p()
        assert self.hip.hipStreamBeginCapture(C.c_void_p(stream), 0) == 0
        work()
        assert self.hip.hipStreamEndCapture(C.c_void_p(stream), C.byref(graph)) == 0
        assert self.hip.hipGraphInstantiate(C.byref(run), graph, None, None, C.c_size_t(0)) == 0
        return run

    def replay(self, run, stream):
        assert self.hip.hipGraphLaunch(run, C.c_void_p(stream)) == 0


@pytest.mark.gpu
def test_captured_and_beside_each_other():
    """two passes on two streams with scratch of their own, and the whole step in a graph that is replayed with eager work between: the same bits each time"""
    U, lib = gpu()
    rng = np.random.default_rng(6)
    hip = Hip()
    passes, streams = [], [hip.stream() for _ in range(2)]
    for seed in range(2):
        q, k, v, seen = inputs(rng, 16, 2, 128, 20, 900, 130)
        p = Pass(U, lib, q, k, v, seen, 900, 0.09)
        x = rng.standard_normal((20, 50000)).astype(np.float32) * 3
        p.x, p.u, p.tk, p.tp = U.Dev(x), U.Dev(rng.random(20).astype(np.float32)), U.Dev(np.array([0, 50] * 10, np.int32)), U.Dev(np.full(20, 0.9, np.float32))
        p.size = lib.pi_op_sample_scratch_bytes(50000, 20)
        p.room_s, p.id, p.prob, p.kept = U.Dev(nbytes=p.size + 16), *[U.Dev(np.zeros(20, np.int32)) for _ in range(3)]
        p.mass, p.source = U.Dev(np.zeros(1030, np.float32)), U.Dev(np.zeros(500, np.int32))
        passes.append(p)

    def step(p, stream):
        p.attend(stream)
        p.give(p.mass, 0.0, stream)
        L.check(lib.pi_op_cache_choose(p.mass.ptr, None, 1030, 500, p.source.ptr, stream), "pi_op_cache_choose")
        L.check(lib.pi_op_sample(p.x.ptr, 50000, 50000, 20, None, p.tk.ptr, p.tp.ptr, None, p.u.ptr, p.room_s.ptr, p.size, p.id.ptr, p.prob.ptr, p.kept.ptr, stream), "pi_op_sample")

    def results(p):
        out, lse = p.outputs()
        return [out, lse, p.mass.get(np.float32), p.source.get(np.int32), p.id.get(np.int32), p.prob.get(np.float32), p.kept.get(np.int32)]

    alone = []
    for p in passes:
        step(p, None)
        alone.append(results(p))
    L.check(lib.pi_device_sync(), "sync")
    for _ in range(5):
        for p, s in zip(passes, streams):
            step(p, s)
    L.check(lib.pi_device_sync(), "sync")
    for p, want in zip(passes, alone):
        assert all(np.array_equal(a, b) for a, b in zip(results(p), want))
    graph = hip.capture(streams[0], lambda: [step(p, streams[0]) for p in passes])
    for i in range(4):
        for p in passes:                                                 # (what the last replay left is gone)
            for d in (p.out, p.lse, p.mass, p.source, p.id):
                L.check(lib.pi_memset(d.ptr, 0, d.nbytes, None), "memset")
            L.check(lib.pi_memcpy_h2d(p.out.ptr, np.full((p.T, p.os), 7.0, np.float32).ctypes.data_as(C.c_void_p), p.out.nbytes, None), "h2d")
        L.check(lib.pi_device_sync(), "sync")
        hip.replay(graph, streams[0])
        L.check(lib.pi_device_sync(), "sync")
        for p, want in zip(passes, alone):
            assert all(np.array_equal(a, b) for a, b in zip(results(p), want)), i
        step(passes[i % 2], None)
        L.check(lib.pi_device_sync(), "sync")


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [32768, 40000, 40001, 131072])
def test_sample_where_runs_of_ids_are_too_unlikely_to_be_drawn(vocab):
    """hundreds of neighbours whose chances round to nothing one by one but not together: none of them is drawn, and every output is written, whatever u falls on"""
    U, lib = gpu()
    rng = np.random.default_rng(vocab)
    x = np.zeros((8, vocab), np.float32)
    x[0, -1] = 32.0                                                      # 0.22 of a step each, 114 steps in 512 of them
    x[1, -1] = 31.3
    x[2, vocab // 2] = 36.0
    x[3] = 0.3 * rng.standard_normal(vocab); x[3, -3] = 34.0
    x[4, :vocab // 2] = -34.0; x[4, vocab // 2:] = rng.standard_normal(vocab - vocab // 2)
    x[5, -1] = 3.2                                                       # (at a temperature of 0.1 as far)
    x[6, 600] = 3.3; x[6, 700:] = -np.inf
    x[7] = -33.0; x[7, rng.integers(0, vocab, 40)] = rng.standard_normal(40)
    temp = np.array([1, 1, 1, 1, 1, 0.1, 0.1, 1], np.float32)
    for u in (0.0, 2.0 ** -40, 2.0 ** -24, 0.5, 1 - 2.0 ** -24):
        got = run_sample(U, lib, x, vocab, (temp, None, None, None), [u] * 8)
        for t in range(8):
            i, p, n, sure = sampled(x[t], temp[t], 0, np.float32(1.0), np.float32(0.0), np.float32(u))
            assert sure or u == 2.0 ** -40, (u, t)                       # (2^-40: sixteen whole steps, where sums of whole steps leave no doubt)
            assert got[0][t] == i and got[2][t] == n and abs(got[1][t] - p) <= 2.0 ** -23 * p, (t, u, got[0][t], i, got[2][t], n, got[1][t], p)
    # behind a nucleus: of the crowd 3.2 below the largest about a quarter stays
    check_sample(U, lib, x[5:6], vocab, (temp[5:6], None, np.full(1, 0.25), None), [0.0])


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [1000, 32768, 40000, 131075])
def test_sample_at_high_temperatures(vocab):
    """logits hundreds and thousands below the largest, at temperatures at which they are drawn"""
    U, lib = gpu()
    rng = np.random.default_rng(vocab + 1)
    x = -3000.0 * rng.random((6, vocab)).astype(np.float32)
    x[1, ::2] = -np.inf
    x[2, vocab // 2:] -= 1e5
    temp = np.array([800.0, 300.0, 5e4, 1e6, 150.0, 2000.0], np.float32)
    for _ in range(3):
        check_sample(U, lib, x, vocab, (temp, None, None, None), rng.random(6))
    check_sample(U, lib, x, vocab, (temp, None, None, np.full(6, 0.001)), rng.random(6))


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv,dim,tokens", [(4, 4, 64, 4), (8, 1, 128, 2), (8, 2, 80, 70), (300, 300, 8, 65)])
@pytest.mark.parametrize("prompt,above,spread", [(1500, 11.9, 0.0), (8000, 11.2, 0.0), (8000, 11.2, 0.5), (8000, 16.0, 2.0), (32000, 15.0, 0.0), (32000, 16.0, 1.0), (32000, 20.0, 2.0)])
def test_a_cell_that_takes_nearly_all(heads, kv, dim, tokens, prompt, above, spread):
    """one cell far above the others with nothing in its values, in front, behind or between: what the others give is as exact as without it"""
    if heads == 300 and prompt > 8000:
        prompt, above = 4000, above - 2.0
    U, lib = gpu()
    rng = np.random.default_rng(prompt + heads + int(above))
    for at in (0, prompt // 3, prompt - 1):
        q, k, v, seen = inputs(rng, heads, kv, dim, tokens, prompt, 0)
        q[:, :, 1:] = spread * rng.standard_normal(q[:, :, 1:].shape)
        q[:, :, 0] = 4.0
        k, v = k[:prompt], (0.5 + rng.random((prompt, kv, dim))).astype(np.float16)
        k[:, :, 0] = 0.0
        k[at] = 0.0
        k[at, :, 0] = above / 4 * dim ** 0.5
        v[at] = 0.0
        p = Pass(U, lib, q, k, v, seen, prompt, dim ** -0.5)
        p.attend()
        got, lse = p.outputs()
        want, want_lse = np.zeros(got.shape), np.zeros(lse.shape)
        for j in range(heads):
            s = q[:, j].astype(np.float64) @ k[:, j * kv // heads].astype(np.float64).T * dim ** -0.5
            want_lse[:, j] = m = np.log(np.exp(s - s.max(1, keepdims=True)).sum(1)) + s.max(1)
            want[:, j] = np.exp(s - m[:, None]) @ v[:, j * kv // heads].astype(np.float64)
        # (Beside FAR and LSE_FAR: where the others are all equal, a sum that the one cell has made large is rounded the same way at every one of its up to prompt / 32 additions, by up to 2^-24 of it.  Else those go either way)
        same = 0.0 if spread else 2.0 ** -24 * ((prompt + 31) // 32)
        assert np.isfinite(got).all() and np.linalg.norm(got - want) <= (FAR + same) * np.linalg.norm(want) and np.abs(lse - want_lse).max() <= LSE_FAR + same


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv,dim,tokens,prompt,own", [(32, 4, 64, 1, 200, 13), (4, 4, 72, 24, 100, 70), (8, 1, 40, 16, 129, 40), (71, 1, 24, 1, 0, 700), (24, 3, 200, 9, 1, 257), (16, 2, 80, 8, 1000, 0), (2, 1, 256, 3, 40, 0),
                                                             (32, 32, 80, 70, 333, 0), (32, 32, 40, 70, 333, 20), (300, 300, 8, 65, 333, 0), (16, 16, 160, 128, 300, 20)])
def test_keys_of_minus_infinity(heads, kv, dim, tokens, prompt, own):
    """a seen key whose score is minus infinity takes its cell out, and nothing else changes, in heads of every length"""
    U, lib = gpu()
    rng = np.random.default_rng(dim + heads)
    q, k, v, seen = inputs(rng, heads, kv, dim, tokens, prompt, own, loners=tokens > 1)
    q[:, :, 0] = q[:, :, 1] = 0.5 + rng.random((tokens, heads))
    for i, c in enumerate(rng.permutation(np.flatnonzero(seen.any(0)))[:4]):
        k[c, :, i % 2] = -np.inf
    want, want_lse, w = soft_max(q, k, v, seen, dim ** -0.5)
    assert np.isfinite(want).all() and np.isfinite(want_lse).any()
    p = Pass(U, lib, q, k, v, seen, prompt, dim ** -0.5)
    p.attend()
    got, lse = p.outputs()
    check_attention(got, want, lse, want_lse)
    p.lse = U.Dev(want_lse.astype(np.float32))
    mass = U.Dev(np.zeros(prompt + own, np.float32))
    p.give(mass, 0.0)
    assert np.allclose(mass.get(np.float32), w.sum((0, 1))[:prompt + own], rtol=8e-6, atol=1e-12)


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv,dim,tokens,prompt,own", [(32, 4, 64, 1, 200, 13), (4, 4, 128, 24, 100, 70), (8, 1, 40, 16, 129, 40), (71, 1, 72, 1, 0, 700), (24, 3, 24, 9, 1, 257), (16, 2, 80, 8, 1000, 0), (2, 1, 256, 3, 40, 0),
                                                             (32, 32, 80, 70, 333, 0), (32, 32, 40, 70, 333, 20), (300, 300, 8, 65, 333, 0), (16, 16, 160, 128, 300, 20)])
def test_values_of_infinity(heads, kv, dim, tokens, prompt, own):
    """an infinite value that a token sees makes an infinity of its output, two of different signs no number; the other outputs are what they are without.  The same where the device says how many cells there are, and without a mask"""
    U, lib = gpu()
    rng = np.random.default_rng(dim + heads + 1)
    q, k, v, seen = inputs(rng, heads, kv, dim, tokens, prompt, own, loners=tokens > 1)
    n = prompt + own
    cells = rng.permutation(np.flatnonzero(seen.any(0)))[:5]
    for c, value in zip(cells, (np.inf, -np.inf, np.inf, -np.inf, np.nan)):
        v[c, rng.integers(0, kv), rng.integers(0, dim, 2)] = value
    v[cells[0], 0, 3], v[cells[1], 0, 3] = np.inf, -np.inf               # both
    rooms = [None, (prompt + 600, n + 900)]
    for room in rooms + ([(n, n)] if own == 0 else []):
        if room:
            k, v = (np.concatenate([x, np.full((max(0, room[1] - len(x)), kv, dim), np.nan, np.float16)]) for x in (k, v))
        with np.errstate(invalid="ignore"):
            want, want_lse, _ = soft_max(q, k, v, seen, dim ** -0.5)
        fine = np.isfinite(want)
        assert np.isinf(want).any() and fine.any()
        p = Pass(U, lib, q, k, v, seen, prompt, dim ** -0.5, room)
        if room == (n, n):
            p.mask.ptr = None
        p.attend()
        got, lse = p.outputs()
        for kind in (np.isposinf, np.isneginf, np.isnan):
            assert (kind(got) == kind(want)).all(), kind
        check_attention(np.where(fine, got, 0), np.where(fine, want, 0), lse, want_lse)


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv,dim,tokens,prompt,own", [(4, 4, 64, 5, 300, 0), (8, 2, 80, 40, 700, 60), (16, 1, 128, 9, 0, 300), (71, 1, 64, 2, 65, 90)])
def test_mass_of_rows_that_give_nothing(heads, kv, dim, tokens, prompt, own):
    """rows of a padded batch: their lse is minus infinity, and whatever their queries hold is without effect; so is a key whose score is minus infinity"""
    U, lib = gpu()
    rng = np.random.default_rng(heads + dim)
    q, k, v, seen = inputs(rng, heads, kv, dim, tokens, prompt, own)
    n, scale = prompt + own, dim ** -0.5
    q[:, :, 0] = 0.5 + rng.random((tokens, heads))
    k[int(np.flatnonzero(seen[0])[0]), :, 0] = -np.inf
    with np.errstate(invalid="ignore"):
        _, want_lse, w = soft_max(q, k, v, seen, scale)
    off = np.zeros((tokens, heads), bool)
    off[tokens // 2] = True
    off[-1, ::2] = True
    want_lse[off], w[off] = -np.inf, 0.0
    q[off] = np.array([np.nan, np.inf, -np.inf, 6e4], np.float16)[rng.integers(0, 4, off.sum())][:, None]
    p = Pass(U, lib, q, k, v, seen, prompt, scale)
    p.lse = U.Dev(want_lse.astype(np.float32))
    old = rng.random(n).astype(np.float32)
    mass = U.Dev(old)
    p.give(mass, 0.5)
    assert np.allclose(mass.get(np.float32), 0.5 * old.astype(np.float64) + w.sum((0, 1))[:n], rtol=8e-6, atol=1e-12)


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [20000, 40000])
def test_sample_between_equal_logits(vocab):
    """equal logits, a border or u between two of them: the one that is drawn is the one by the definition or its neighbour among those that stay"""
    U, lib = gpu()
    x = np.zeros((4, vocab), np.float32)
    x[1, ::3] = 1.0
    x[2, 1::2] = -np.inf
    x[3, :100] = 5.0
    for u in (0.0, 0.25, 0.3, 0.5, 0.777, 1 - 2.0 ** -24):
        for k, top_p in ((0, 1.0), (100, 1.0), (0, 0.5), (777, 0.4321), (5000, 0.75)):
            got = run_sample(U, lib, x, vocab, (None, np.full(4, k), np.full(4, top_p), None), [u] * 4)
            for t in range(4):
                i, _, n, _ = sampled(x[t], np.float32(1.0), k, np.float32(top_p), np.float32(0.0), np.float32(u))
                ids = np.flatnonzero(x[t] > -np.inf)
                ids = np.sort(ids[np.argsort(-x[t, ids], kind="stable")][:n + 1])      # (the next one may stay, where a border is a whole count)
                assert abs(int(got[2][t]) - n) <= 1 and got[0][t] in ids and abs(int(np.searchsorted(ids, got[0][t])) - int(np.searchsorted(ids, i))) <= 1, (t, u, k, top_p, got[0][t], i, got[2][t], n)


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv,dim,tokens,prompt,out", [(300, 300, 8, 65, 700, 300), (32, 32, 80, 70, 900, 650), (8, 2, 64, 3, 1500, 1100), (4, 1, 128, 40, 700, 500), (16, 16, 64, 1, 400, 390)])
def test_a_run_of_keys_of_minus_infinity(heads, kv, dim, tokens, prompt, out):
    """hundreds of cells in front whose scores are minus infinity, and low scores behind them: the first that count come late"""
    U, lib = gpu()
    rng = np.random.default_rng(out)
    for low in (15.0, 40.0, 80.0):
        q, k, v, seen = inputs(rng, heads, kv, dim, tokens, prompt, 0)
        q[:, :, 0] = q[:, :, 1] = 4.0
        k[:out, :, 0] = -np.inf
        k[out:prompt, :, 1] = -low / 4 * dim ** 0.5
        k, v = k[:prompt], (0.5 + rng.random((prompt, kv, dim))).astype(np.float16)
        want, want_lse, _ = soft_max(q, k, v, seen, dim ** -0.5)
        p = Pass(U, lib, q, k, v, seen, prompt, dim ** -0.5)
        p.attend()
        got, lse = p.outputs()
        # (scores of up to 2^7 in powers of two: a sum of products is rounded once for every sixteen of them, the scale, its product with a score and the difference once each, every time by up to 2^-24 of the score: so much x ln 2 of a
        # weight and of the lse)
        far = ((dim + 15) // 16 + 3) * 2.0 ** -17 * np.log(2)
        assert np.isfinite(got).all() and np.linalg.norm(got - want) <= far * np.linalg.norm(want) and np.abs(lse - want_lse).max() <= far


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv,dim,tokens,prompt", [(300, 300, 8, 65, 700), (8, 2, 64, 3, 1500), (4, 4, 128, 1, 333), (16, 16, 64, 40, 900)])
def test_equal_scores(heads, kv, dim, tokens, prompt):
    """every cell the same weight, whatever the score: the mean of the values"""
    U, lib = gpu()
    rng = np.random.default_rng(prompt)
    for score in (-11.0, -7.0, -5.0, -4.5, -2.0, -0.6, 0.0, 1.9, 3.3, 8.0, 30.0):
        q, k, v, seen = inputs(rng, heads, kv, dim, tokens, prompt, 0)
        q[:] = 0.0
        q[:, :, 0] = 2.0
        k, v = np.zeros((prompt, kv, dim), np.float16), (0.5 + rng.random((prompt, kv, dim))).astype(np.float16)
        k[:, :, 0] = score / 2 * dim ** 0.5
        p = Pass(U, lib, q, k, v, seen, prompt, dim ** -0.5)
        p.attend()
        got, lse = p.outputs()
        want = np.repeat(v.astype(np.float64).mean(0), heads // kv, axis=0)[None]
        # (The sum of the weights is rounded the same way at every one of its up to prompt / 32 additions, by 2^-24 of it at most; a weight and its two halves differ by 2^-23; the sums of the products go either way.  lse: at most 2^6, the score as in FAR)
        far = 2.0 ** -24 * ((prompt + 31) // 32) + 2.0 ** -22
        assert np.abs(got / want - 1).max() <= far and np.abs(lse - (2.0 * k[0, 0, 0].astype(np.float64) * dim ** -0.5 + np.log(prompt))).max() <= LSE_FAR, (score, np.abs(got / want - 1).max(), far)


def test_scales_that_powers_of_two_do_not_hold():
    """scores are taken in powers of two: a scale that is infinite there is refused, not answered with no numbers"""
    lib = L.load()
    for scale in (2.4e38, 3.4e38):
        assert attention_call(lib, scale=scale) != 0 and b"scale" in lib.pi_last_error()
        assert lib.pi_op_attention_mass(P, 512, P, P, P, scale, 64, 8, 2, 3, 100, 140, 1.0, P, 1 << 40, P, None, None) != 0 and b"scale" in lib.pi_last_error()
