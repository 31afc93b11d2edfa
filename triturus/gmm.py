"""Import path beside the reference's modules: ``from triturus.gmm import gmm, gmm_grad``."""
from triturus_amd.gmm import gmm, gmm_grad  # noqa: F401
