"""A layer's device step, without a GPU: what its attention would refuse is refused before anything is launched, so that no token
is stored by a step that fails."""

import threading
import types

import pytest

from tests.test_attention_numbers_host import A, Calls
from vesper_amd.attention import CachedAttention, rotation_table
from vesper_amd.projections import FP8_LAYOUT


class Opened(Calls):
    """A context on which a layer can be opened, and nothing run."""

    def upload(self, *_):
        return self.empty()

    def fp8_reserve(self, *_):
        pass


@pytest.mark.parametrize("change", [dict(tokens=3), dict(batch=0), dict(columns=0), dict(columns=2 ** 26 + 1), dict(columns=2 ** 32 + 1), dict(table_ptr=None),
                                    dict(table_ptr=0), dict(lengths_ptr=None), dict(table_ptr=A + 2), dict(lengths_ptr=A + 1),
                                    dict(q_first_ptr=A + 2), dict(tokens=5), dict(batch=5), dict(tokens=-1), dict(batch=-1)])
def test_refused_before_anything_runs(change):
    def project(*_, **__):
        pytest.fail("a refused step projected")
    runtime = types.SimpleNamespace(ctx=Opened(), block=32, has_wo_a=True, layout=dict(FP8_LAYOUT), project_device=project, _ready=lambda: None,
                                    tiled={"wo_a": A}, lock=threading.Lock())
    layer = CachedAttention(runtime, 4, 16, rotation_table(8, 64), max_tokens=4, max_batch=4)
    args = dict(x_ptr=A, tokens=4, positions_ptr=A, slots_ptr=A, table_ptr=A, columns=1, lengths_ptr=A, batch=2, y_ptr=A)
    with pytest.raises(ValueError):
        layer.step_device(**{**args, **change})
