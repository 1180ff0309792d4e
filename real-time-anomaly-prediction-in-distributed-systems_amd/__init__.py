"""MI355X-native batched HTM engine (encoder -> SP -> BacktrackingTM -> anomaly).

Import through the repo-root helper `_pkg.load()` (the package directory name
is not a Python identifier); it registers this package as `rtap_amd`.
"""
from . import _lib
from ._lib import HtmConfig, HtmError, build, default_config
from .engine import HTMEngine
from . import classifier, fleet, harness, ingest
from .beam import beam_reorder, beam_select
from .harness import AnomalyLikelihood, SLOHarness
from .network import BatchRecordStream, MultiEncoder, Network, ScalarEncoder
from .readout import Readout4

__all__ = ["AnomalyLikelihood", "SLOHarness", "HTMEngine", "Network", "BatchRecordStream", "MultiEncoder", "ScalarEncoder", "HtmConfig", "HtmError", "Readout4", "beam_reorder", "beam_select", "build", "default_config", "_lib"]
