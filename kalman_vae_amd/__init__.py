"""MI355X-native Kalman filter / RTS smoother / Kalman-ELBO hot path of the
Kalman VAE, behind the reference's ``StateSpaceModel`` interface.

Compute runs only in the HIP library kalman_vae_amd/csrc/libkvae_kalman.so
(gfx950); there is no CPU implementation in this package.
"""
from .sample_control import SampleControl
from .misc import aggregate
from .dynamics_parameter_network import GatedModel, LSTMModel, MLPModel
from .state_space_model import StateSpaceModel
from .elbo import kalman_elbo
from .variational_autoencoder import BernoulliDecoder, Encoder, GaussianDecoder
from .kalman_vae import KalmanVariationalAutoencoder
from .sequence_ops import (gated_scan, gated_scan_step, linear_8bit, quantize_rows, rms_norm,
                           rms_norm_quantized)
from .optim import AdamW, adamw_step
from .functions import (kalman_filter_steps, kalman_smooth_steps, kalman_elbo_terms,
                        read_status)

__all__ = ["SampleControl", "aggregate", "GatedModel", "LSTMModel", "MLPModel",
           "StateSpaceModel",
           "kalman_elbo", "KalmanVariationalAutoencoder", "Encoder", "GaussianDecoder",
           "BernoulliDecoder", "kalman_filter_steps", "kalman_smooth_steps", "kalman_elbo_terms",
           "read_status", "gated_scan", "gated_scan_step", "rms_norm",
           "rms_norm_quantized", "quantize_rows", "linear_8bit", "AdamW", "adamw_step"]
