"""The example's command takes two words and no others: a misspelt one trained another model."""

import pytest

import sequence


@pytest.mark.parametrize("words", [("rewards",), ("Delta", "reward"), ("delta", "")])
def test_unknown_words(tmp_path, words):
    with pytest.raises(ValueError, match="delta and reward"):
        sequence.main(str(tmp_path), 1, *words)
