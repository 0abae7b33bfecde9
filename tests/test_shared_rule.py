"""``config.shared_prefix_pays``: which fused layer steps take a plan of shared prefixes (no GPU)."""

from types import SimpleNamespace

from oscar_new_amd.backend import OscarAttentionImpl
from oscar_new_amd.config import shared_prefix_pays as pays

# (requests, query tokens each, shared, length), measured without and with the plan (us).
FASTER_WITH = [(96, 1, 16000, 16650), (256, 1, 32000, 32650), (64, 1, 64000, 64650),
               (256, 1, 12000, 16000), (8, 4, 100, 2000), (16, 2, 32000, 32650),
               (160, 3, 8000, 16000), (2, 64, 32000, 32700), (4, 64, 16000, 16700)]
SLOWER_WITH = [(6, 1, 2000, 2500), (2, 1, 128000, 128600), (32, 1, 32000, 32650),
               (64, 1, 4000, 16000), (128, 1, 8000, 32000), (160, 3, 800, 16000),
               (24, 8, 3200, 64000), (2, 256, 32000, 32900), (8, 64, 3200, 64000)]


def test_choices_of_measured_steps():
    for steps, want in ((FASTER_WITH, True), (SLOWER_WITH, False)):
        for members, n, share, length in steps:
            args = (members * n, members, 1, n, members * length)
            assert pays(*args, saved_tokens=(members - 1) * share) is want, (members, n, share)


def test_unknown_lengths_and_savings():
    assert pays(4, 4, 1, 1) and pays(256, 64, 1, 4)  # a capture of dummy lengths
    assert pays(100, 100, 1, 1, saved_tokens=2_000_000)
    assert not pays(100, 100, 1, 1, saved_tokens=1_000_000)
    # At best: one group that shares everything.
    assert pays(100, 100, 1, 1, 3_000_000) and not pays(100, 100, 1, 1, 1_300_000)
    assert pays(100, 100, 2, 1, 1_300_000)  # as many positions again of the second KV head


def test_a_layer_asks_the_rule():
    impl = OscarAttentionImpl.__new__(OscarAttentionImpl)
    impl.num_kv_heads = 1
    meta = SimpleNamespace(max_query_len=1, num_reqs=256, total_seq_len=256 * 16000, shared=None)
    assert not impl._takes_shared(meta, 256)
    meta.shared = SimpleNamespace(saved_tokens=None)
    assert impl._takes_shared(meta, 256)
    meta.shared.saved_tokens = 255 * 4000
    assert not impl._takes_shared(meta, 256)
    del meta.total_seq_len
    meta.shared.saved_tokens = None
    assert impl._takes_shared(meta, 256)
