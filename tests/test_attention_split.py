"""CPU: the scratch of the attention backward under STEW_ATTN_SPLIT."""
import pytest

CAP = 4096 * 128 * 256 * 4  # key tiles x shares, 128 rows of [dK | dV] in fp32


def _bytes(tokens, heads, kv_heads, head_dim=128, rows=1):
    from stew_b200 import _lib
    a = _lib.AttnC()
    a.q = a.k = a.v = a.cu = 256
    a.tokens, a.rows, a.heads, a.kv_heads, a.head_dim = tokens, rows, heads, kv_heads, head_dim
    a.q_stride, a.q_head_stride = heads * head_dim, head_dim
    a.k_stride = a.v_stride = kv_heads * head_dim
    a.k_head_stride = a.v_head_stride = head_dim
    a.dtype, a.left, a.right, a.scale = _lib.NF4B_F16, -1, 0, 0.125
    return _lib.lib().nf4b_attn_bwd_work_bytes(bytes(a))


def _unshared(tokens, heads, kv_heads, rows=1):
    """Rows' (lse, delta), tiles' maxima, tickets: what one share needs, rounded up."""
    slots = tokens // 128 + rows + 1
    return heads * tokens * 8 + heads * slots * 8 + 2 * slots * kv_heads * 4 + 5 * 16


@pytest.mark.parametrize("tokens,heads,kv_heads,split", [(1 << 20, 12, 2, "6"), (1 << 20, 12, 2, "2"), (300_000, 8, 1, "8"),
                                                         (200_000, 16, 16, "1"), (131_072, 9, 1, "9"), (120_000, 12, 2, "3")])
def test_an_override_keeps_the_scratch_within_the_cap(monkeypatch, tokens, heads, kv_heads, split):
    monkeypatch.setenv("STEW_ATTN_SPLIT", split)
    assert 0 < _bytes(tokens, heads, kv_heads) <= _unshared(tokens, heads, kv_heads) + CAP


def test_an_override_within_the_cap_holds(monkeypatch):
    sizes = []
    for split in ("1", "2", "3", "6"):
        monkeypatch.setenv("STEW_ATTN_SPLIT", split)
        sizes.append(_bytes(1170, 12, 2, rows=4))
    pairs = (1170 // 128 + 5) * 2
    assert sizes[0] <= _unshared(1170, 12, 2, rows=4)
    assert [s - sizes[0] for s in sizes[1:]] == [pairs * n * 128 * 256 * 4 for n in (2, 3, 6)]
    monkeypatch.setenv("STEW_ATTN_SPLIT", "5")  # no divisor of the group
    ignored = _bytes(1170, 12, 2, rows=4)
    monkeypatch.delenv("STEW_ATTN_SPLIT")
    assert ignored == _bytes(1170, 12, 2, rows=4)
