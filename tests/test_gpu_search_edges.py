"""Edges of the generator's search: none, one and no more bytes."""
from __future__ import annotations

import pytest

from leo_amd import native
from leo_amd.generate import Generator
from leo_amd.model import Model
from leo_amd.runtime import HipRuntime
from tests.helpers import small_redundant_config

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("count", [0, -3, 1, 2])
def test_the_document_has_ended_after_any_search(require_gpu, count):
    with HipRuntime(Model.synthetic(small_redundant_config(), weight_sigma=0.05), max_lanes=1) as runtime:
        generator = Generator(runtime)
        generator.prompt(b"the ")
        found = generator.search(count, beams=3)
        assert found == [(b"", 0.0)] if count < 1 else len(found) == 3
        for call in (lambda: generator.search(count), lambda: generator.write(2)):
            with pytest.raises(native.LeoError) as err:
                call()
            assert err.value.code == native.ERR_INVALID_ARGUMENT and "document" in str(err.value)
        generator.prompt(b"the ")
        assert len(generator.write(2, allow_end=False)[0]) == 2
