"""The kernels and refusals of the caller-owned paged cache on the CPU emulation (bounds-checked by AddressSanitizer,
pages bit for bit, attention within its derived bound; no GPU needed)."""
import os

import pytest

from tests.hipemu import runner
from tests.test_hipemu import emu_lib  # noqa: F401

ORDER = ["paged_shared_int8", "paged_shared_int4", "paged_shared_fp16", "paged_chunks", "paged_rows", "paged_refusals"]


@pytest.fixture(scope="module")
def runs(emu_lib):  # noqa: F811
    pool = runner.ScenarioPool(ORDER, jobs=max(1, min(6, (os.cpu_count() or 2) - 2)))
    yield pool
    pool.close()


@pytest.mark.parametrize("name", ORDER)
def test_paged(runs, name):
    assert runs.result([name], timeout=1800) == 0
