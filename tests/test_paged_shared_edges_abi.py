"""mx_paged_decode_shared on the CPU: sizes at the ends of what it takes."""
from dooms_amd import _lib
from dooms_amd import attention as A


def test_a_size_that_succeeds_leaves_the_last_error():
    """More (kv head, row tile) pairs than a decode counts: only a call without groups is one."""
    size = lambda n_groups: A.paged_shared_workspace_bytes(n_head=4096, n_head_kv=4096, head_dim=64, n_q=1, n_seq=4, n_groups=n_groups, max_own_len=100)
    assert _lib.paged_decode_shared_workspace_bytes(_lib.MxPagedDesc(n_head=1, n_head_kv=1, head_dim=96, dtype=_lib.DTYPE_F16), 1) == 0
    before = _lib.last_error()
    assert "head_dim" in before
    assert size(1) > 0 and _lib.last_error() == before
    assert size(0) == 0 and "more than one launch" in _lib.last_error()


def test_as_many_groups_as_sequences():
    """At the most of both, as with half the groups."""
    size = lambda n_groups, n_kv: A.paged_shared_workspace_bytes(n_head=n_kv, n_head_kv=n_kv, head_dim=64, n_q=1, n_seq=65535, n_groups=n_groups,
                                                                 max_own_len=100)
    for n_kv in (1, 64, 120):
        assert size(65535, n_kv) >= size(32767, n_kv) > 0
    assert size(65535, 256) == 0 and "more than one launch" in _lib.last_error()
