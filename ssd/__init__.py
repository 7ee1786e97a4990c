"""Makes ``import ssd`` work from the repository's root: the package is subnetwork-speculative-decoding_amd/ssd, whose __init__ runs here."""

import os

__path__ = [os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "subnetwork-speculative-decoding_amd", "ssd")]
with open(os.path.join(__path__[0], "__init__.py")) as _f:
    exec(compile(_f.read(), _f.name, "exec"))
