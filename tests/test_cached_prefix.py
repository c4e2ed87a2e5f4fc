"""The attention mode of requests behind a cached prefix, on the CPU."""
import warnings

import pytest


def test_auto_of_the_prefix_and_of_the_whole_request(pkg):
    """AUTO is resolved on the prefix; where the whole request would run in the other
    mode, the caller hears of it."""
    full, sparse = pkg.attention.MODE_FULL, pkg.attention.MODE_SPARSE
    prefix = pkg.model.CachedPrefix(5000, sparse, [], auto=True)
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        for longest in (0, 1, 3192):
            assert prefix.mode_for(longest) == sparse
        assert pkg.model.CachedPrefix(9000, full, [], auto=True).mode_for(100) == full
        assert pkg.model.CachedPrefix(5000, sparse, []).mode_for(4000) == sparse  # was asked for
    for longest in (3193, 4000):
        with pytest.warns(UserWarning, match="MODE_FULL"):
            assert prefix.mode_for(longest) == sparse
