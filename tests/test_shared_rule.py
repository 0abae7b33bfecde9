"""``config.shared_prefix_pays``: which fused layer steps take a plan of shared prefixes (no GPU)."""

from types import SimpleNamespace

from oscar_new_amd.backend import OscarAttentionImpl
from oscar_new_amd.config import OscarConfig, shared_prefix_pays as pays

# (KV heads, heads each, groups, members, shared tokens, query tokens, all tokens), measured step
# without and with the plan (us).
STEPS = [((1, 6, 1, 2, 32000, 1, 65273), 26.6, 34.4), ((1, 6, 1, 32, 32000, 1, 1044773), 43.3, 47.6),
         ((1, 6, 1, 96, 64000, 1, 6206321), 188.9, 108.0), ((1, 6, 1, 64, 4000, 1, 1024000), 51.1, 67.2),
         ((1, 6, 1, 256, 32000, 1, 8358199), 214.3, 127.9), ((1, 6, 1, 128, 8000, 1, 4096000), 130.3, 178.3),
         ((1, 6, 1, 16, 128000, 2, 2058398), 112.4, 76.2), ((1, 6, 1, 160, 800, 3, 2559974), 182.5, 237.8),
         ((1, 6, 1, 192, 32000, 4, 6269133), 409.0, 247.2), ((1, 6, 1, 24, 3200, 8, 1535996), 179.9, 231.8),
         ((1, 6, 1, 8, 128000, 16, 1029287), 220.6, 160.0), ((1, 6, 8, 8, 32000, 1, 2089488), 78.0, 64.7),
         ((1, 6, 1, 2, 32000, 256, 65850), 198.8, 221.8), ((1, 6, 1, 8, 3200, 64, 511996), 314.3, 380.6),
         ((2, 4, 1, 4, 1500, 2, 8000), 26.4, 34.3), ((2, 6, 1, 4, 60000, 64, 255996), 319.3, 394.8),
         ((4, 8, 1, 8, 800, 4, 127996), 82.2, 98.9), ((4, 8, 1, 64, 8000, 4, 1024000), 279.3, 321.1)]


def choice(heads, group, groups, members, shared, queries, total, **over):
    reqs = groups * members
    args = dict(total_seq_len=total, saved_tokens=groups * (members - 1) * shared, groups=groups)
    return pays(reqs * queries, reqs, heads, heads * group, queries, **dict(args, **over))


def test_no_measured_step_gets_slower_and_the_large_gains_are_taken():
    for step, without, with_plan in STEPS:
        assert choice(*step) is (with_plan < 0.85 * without), step
        assert choice(*step, total_query_keys=step[5] * step[6]) is choice(*step)


def test_unknown_lengths_and_savings():
    few, many = STEPS[0][0], STEPS[4][0]
    assert choice(*few, total_seq_len=None) and choice(*many, total_seq_len=None)
    assert choice(*many, saved_tokens=None) and not choice(*few, saved_tokens=None)
    assert not choice(*many, saved_tokens=1_000_000)
    assert not pays(256, 256, 1, 6, 1, 8358199, groups=256) and not choice(*many, saved_tokens=0)
    assert not pays(1, 1, 1, 6, 1, 100_000_000)


def test_a_layer_asks_the_rule():
    impl = OscarAttentionImpl.__new__(OscarAttentionImpl)
    impl.num_kv_heads, impl.num_heads = 1, 6
    meta = SimpleNamespace(max_query_len=1, num_reqs=256, total_seq_len=256 * 16000, shared=None,
                           layout=SimpleNamespace(config=OscarConfig()))
    assert not impl._takes_shared(meta, 256)
    meta.shared = SimpleNamespace(saved_tokens=None, groups=1)
    assert impl._takes_shared(meta, 256)
    meta.shared.saved_tokens = 255 * 4000
    assert not impl._takes_shared(meta, 256)
    del meta.total_seq_len
    assert impl._takes_shared(meta, 256)
