"""What the paged-cache entry points refuse before any launch, through the C ABI on a machine without a GPU."""
from merak_amd import _lib

A = 4096          # an aligned address that no call gets as far as using


def err():
    return _lib.lib().mtp_last_error().decode()


def test_paged_plan_refusals():
    f = _lib.lib().mtp_paged_plan
    ok = dict(requests=2, max_pages=4, page=16, free=8, tokens=3)

    def call(ptrs=(A,) * 11 + (A + 64, A + 64), **over):
        s = {**ok, **over}
        return f(*ptrs, s["requests"], s["max_pages"], s["page"], s["free"], s["tokens"], None)

    assert call(page=24) == -1 and "power of two" in err()
    assert call(page=0) == -1
    assert call(requests=4097) == -2 and "4097" in err()
    assert call(requests=-1) == -2
    assert call(max_pages=0) == -1 and call(free=-1) == -1 and call(tokens=-1) == -1 and call(tokens=2 ** 31) == -1
    assert call(max_pages=2 ** 28, page=16) == -1                       # a row of 2^32 tokens
    assert call(ptrs=(A,) * 12 + (A + 64,)) == -1 and "share" in err()   # held in place
    assert call(ptrs=(A,) * 11 + (A + 64, A)) == -1 and "share" in err()
    for i in (0, 1, 2, 3, 4, 5, 6, 7, 8, 9, 10, 11, 12):
        p = [A] * 11 + [A + 64, A + 64]
        p[i] = None
        assert call(ptrs=tuple(p)) == -1 and "null" in err(), i
    r = _lib.lib().mtp_paged_release
    assert r(None, A, A, A, A, 2, 4, 8, None) == -1 and r(A, A, A, A, A, 5000, 4, 8, None) == -2
    assert r(None, None, None, None, None, 0, 4, 8, None) == 0


def test_qk_norm_rope_refusals():
    lib = _lib.lib()

    def fwd(T=2, nq=2, nk=1, d=128, P=10, dtype=1, table=0, p=(A,) * 8):
        return lib.mtp_qk_norm_rope(p[0], p[1], p[2], table, p[3], p[4], p[5], p[6], p[7], T, nq, nk, d, P, 1e-6, dtype, None)

    assert fwd(d=96) == -2 and "96" in err()
    assert fwd(dtype=5) == -1 and fwd(table=2) == -1 and "tables" in err()
    assert fwd(T=-1) == -1 and fwd(nq=0) == -1 and fwd(nk=0) == -1 and fwd(P=0) == -1 and fwd(T=2 ** 22) == -2
    assert fwd(p=(A + 2,) + (A,) * 7) == -1 and "aligned" in err()
    assert fwd(p=(None,) + (A,) * 7) == -1 and fwd(p=(A,) * 6 + (None, A)) == -1 and fwd(p=(A,) * 3 + (None,) + (A,) * 4) == -1
    assert fwd(T=0, p=(None,) * 8) == 0

    def app(dtype=1, pages=4, page=16, slots=A, T=2):
        return lib.mtp_qk_norm_rope_append(A, A, A, 0, A, slots, None, None, A, A, A, T, 2, 1, 128, 10, pages, page, 1e-6, dtype,
                                           None)

    assert app(dtype=0) == -2 and app(page=3) == -1 and app(pages=0) == -1 and app(slots=None) == -1 and app(T=0) == 0

    def bwd(dqw=A, qw=A, ws=A, wsb=1 << 30, T=2, dqkv=A):
        return lib.mtp_qk_norm_rope_bwd(A, A, A, A, A, A, 0, A, qw, None, dqkv, dqw, None, ws, wsb, T, 2, 1, 128, 10, 1e-6, 1, None)

    need = lib.mtp_qk_norm_rope_bwd_workspace_bytes(2, 2, 1, 128)
    assert need > 0 and lib.mtp_qk_norm_rope_bwd_workspace_bytes(2, 2, 1, 80) == 0
    assert bwd(qw=None) == -1 and "without its weight" in err()
    assert bwd(ws=None) == -4 and bwd(wsb=need - 1) == -4 and bwd(dqkv=None) == -1
    assert bwd(T=0) == -1 and bwd(T=0, dqw=None) == 0


def test_attn_paged_refusals():
    lib = _lib.lib()
    full = lib.mtp_attn_paged_workspace_bytes()
    assert 4096 < full < 1 << 28

    def call(p=(A,) * 8, wsb=full, T=3, R=2, nq=8, nk=2, d=128, pages=9, page=16, row=4, new=1, bound=64, scale=0.1, dtype=1):
        return lib.mtp_attn_paged(*p, wsb, T, R, nq, nk, d, pages, page, row, new, bound, scale, dtype, None)

    assert call(dtype=0) == -2 and call(d=96) == -2 and call(nq=7) == -1 and call(nk=0) == -1
    assert call(page=8) == -2 and call(page=48) == -2 and "48" in err()
    assert call(pages=0) == -1 and call(row=0) == -1 and call(row=2 ** 27) == -1 and call(T=2 ** 30) == -1
    assert call(new=-1) == -1 and call(bound=-1) == -1
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        assert call(scale=scale) == -1 and "scale" in err()
    assert call(wsb=full - 1) == -4
    for i in range(7):
        p = [A] * 8
        p[i] = None
        assert call(p=p) == -1 and "null" in err(), i
    assert call(p=[A] * 7 + [None]) == -4
    for i in (0, 1, 2, 6, 7):
        p = [A] * 8
        p[i] = A + 8
        assert call(p=p) == -1 and "aligned" in err(), i
    assert call(T=0, p=(None,) * 8) == 0 and call(R=0, p=(None,) * 8) == 0


def test_verify_draft_refusals():
    lib = _lib.lib()
    need = lib.mtp_verify_draft_workspace_bytes(2, 1000)
    assert need > 0 and lib.mtp_verify_draft_workspace_bytes(0, 1000) == 0

    def call(p=(A, None, A, None, A, A, A), ws=A, wsb=need, R=2, K=3, V=1000, dtype=0):
        return lib.mtp_verify_draft(*p, ws, wsb, R, K, V, dtype, None)

    assert call(dtype=9) == -1 and call(V=0) == -1 and call(R=65536) == -1 and call(R=-1) == -1
    assert call(K=65) == -2 and "65" in err() and call(K=-1) == -2
    assert call(ws=None) == -4 and call(wsb=need - 1) == -4 and call(ws=A + 4) == -4
    for i in (0, 2, 4, 5, 6):
        p = [A, None, A, None, A, A, A]
        p[i] = None
        assert call(p=p) == -1, i
    assert call(R=0, p=(None,) * 7, ws=None, wsb=0) == 0
