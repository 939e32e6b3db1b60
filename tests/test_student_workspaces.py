"""The workspaces that a student's operators ask for: 0 where no call takes the sizes, and never less than their parts."""


def test_sizes_that_no_call_takes(kgx):
    L, over, top = kgx.lib(), 2 ** 30 + 1, 2 ** 31 - 1
    for n in (0, -1, -2 ** 31, over, top):
        assert L.kg_distill_loss_workspace(n, 2000, 50) == L.kg_distill_loss_workspace(50, n, 300) == L.kg_distill_loss_workspace(50, 2000, n) == 0
        assert L.kg_layer_norm_workspace(n, 16) == L.kg_layer_norm_workspace(16, n) == 0
        assert L.kg_embedding_backward_workspace(n, 16, 16) == L.kg_embedding_backward_workspace(16, n, 16) == 0
        assert L.kg_embedding_backward_workspace(16, 16, n) == 0
    assert L.kg_distill_loss_workspace(50, 2000, 1025) == 0


def test_largest_sizes_do_not_overflow(kgx):
    L, most = kgx.lib(), 2 ** 30
    assert L.kg_distill_loss_workspace(most, most, 1024) >= most * 1024 * 20
    assert L.kg_layer_norm_workspace(most, most) >= most * 16 + 1024 * 2 * most * 4
    assert L.kg_embedding_backward_workspace(most, most, most) >= most * 8 + most // (64 * 4) * 2 * most * 4
