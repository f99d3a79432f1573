"""Plans of the training attention calls at sizes no test can run: read off the
workspace sizes, which are made of them and need no device."""
import ctypes

import pytest

from tests.test_attention_train_cpu import args, lib


def sizes(with_kv=True, **attn):
    L, n = lib(), ctypes.c_int64(0)
    t = args(dict(prefix_len=-1, dead_start=0, dead_end=0, **attn))
    if not with_kv:
        t.dk = t.dv = None
    out = []
    for f in (L.vlak_attn_gqa_train_workspace_size, L.vlak_attn_gqa_bwd_workspace_size):
        assert f(ctypes.byref(t), ctypes.byref(n)) == 0
        out.append(n.value)
    return out


# A wait in the kernels gives up after a second, and some last a whole item. A step
# of 64 rows or keys takes about half a microsecond, so an item of 2^18 steps takes
# 0.15 s: the most that any may have, however evenly the work would lie otherwise.
MOST = 1 << 18


@pytest.mark.parametrize("log_rows", [24, 25, 26])
def test_no_item_of_keys_outlasts_a_wait(log_rows):
    # one head and many keys, so that the balance alone asks for no parts
    M, N = 1 << log_rows, 1 << 20
    _, bwd = sizes(B=1, M=M, N=N, H=1, Hkv=1)
    statistics, parts = M // 64 * 512 + 256, M // 64 // MOST
    sums = parts * N * 128 * 4 if parts > 1 else 0
    assert bwd == statistics + sums


@pytest.mark.parametrize("log_keys", [24, 25, 26])
def test_no_item_of_rows_outlasts_a_wait(log_keys):
    M, N = 1 << 20, 1 << log_keys
    fwd, bwd = sizes(B=1, M=M, N=N, H=1, Hkv=1, with_kv=False)
    parts = N // 64 // MOST
    assert fwd == (parts * M * (64 * 4 + 8) if parts > 1 else 0)
    assert bwd == M // 64 * 512 + 256 + (parts * M * 64 * 4 if parts > 1 else 0)


def test_many_heads_on_one_kv_head():
    # 2^20 rows of 128 heads on 9600 keys: 2^21 steps for each block of 128 keys
    _, bwd = sizes(B=1, M=1 << 20, N=9600, H=128, Hkv=1)
    assert bwd == (1 << 21) * 512 + 256 + 8 * 75 * 128 * 128 * 4


def test_ordinary_sizes_keep_their_plans():
    # 3 heads of 64 sub-tiles of 64 rows for each kv head (in one box of three
    # heads and 21 positions they would be 196)
    assert sizes(B=2, M=4096, N=4096, H=15, Hkv=5) == [0, 2 * 5 * 3 * 64 * 512 + 256]


# 2^30 rows or keys of one head, twice (q and o, k and v), are 275 GB, and 2^34
# rows in all 2 TB; below them every count of the kernels fits 32 bits
@pytest.mark.parametrize("attn", [dict(M=(1 << 31) - 1, H=1), dict(M=(1 << 30) + 1, H=1),
                                  dict(M=1 << 28, H=128), dict(M=1, N=(1 << 31) - 1, H=1),
                                  dict(M=1, N=(1 << 30) + 1, H=1), dict(M=1, B=1 << 20, N=1 << 15, H=1)])
def test_sizes_whose_counts_pass_32_bits_are_refused(attn):
    L, n = lib(), ctypes.c_int64(0)
    t = args({**dict(B=1, N=64, Hkv=1, prefix_len=-1, dead_start=0, dead_end=0), **attn})
    for f in (L.vlak_attn_gqa_train_workspace_size, L.vlak_attn_gqa_bwd_workspace_size):
        assert f(ctypes.byref(t), ctypes.byref(n)) == 1 and n.value == 0
    assert L.vlak_attn_gqa_train_fwd(ctypes.byref(t), 0x1000, 1 << 60, None) == 1
    assert L.vlak_attn_gqa_bwd(ctypes.byref(t), 0x1000, 1 << 60, None) == 1
    assert b"too many rows or keys" in L.vlak_last_error_message()


def test_the_largest_sizes_have_plans():
    for attn in (dict(M=1 << 30, N=64, H=1, Hkv=1), dict(M=1, N=1 << 30, H=1, Hkv=1),
                 dict(M=1 << 27, N=64, H=128, Hkv=1)):
        fwd, bwd = sizes(B=1, **attn)
        assert 0 <= fwd < 1 << 50 and 0 < bwd < 1 << 50
