"""The embedding, label and gradient operators at the edges of what their documentation allows, ahead of any launch (no
GPU needed)."""
import pytest

P = 0x1000  # a non-null, 16-byte aligned dummy: never dereferenced on these paths
NULL = None


@pytest.mark.parametrize("n", [0, 1, 256, 257, 5000, 1 << 29])
@pytest.mark.parametrize("D", [0, 1, 128, 129])
def test_workspace_of_a_table_without_rows_or_columns(n, D):
    from gsplat import _backend as B

    L = B.lib()
    assert L.gs_embedding_bwd_workspace_bytes(n, 0, D) == 0
    assert L.gs_embedding_bwd(n, 0, D, 0, P, 8, P, D, 1.0, NULL, 0, NULL, NULL) == 0
    for V in (1, 64, 65, 1 << 30):
        assert L.gs_embedding_bwd_workspace_bytes(n, V, 0) == 0
        assert L.gs_embedding_bwd(n, V, 0, 0, P, 8, P, 0, 1.0, NULL, 0, NULL, NULL) == 0
